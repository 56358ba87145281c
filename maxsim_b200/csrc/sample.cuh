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

#include <type_traits>

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

// Order-preserving image of a float; -0 and +0 are equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// 2^y to within 6e-9 of its size, for y <= 0: 2^floor(y + 1/2) times the Taylor series of
// e^r at r = ln 2 (y - floor(y + 1/2)), |r| <= 0.3466, cut after r^7 / 7! (the next
// term is 0.3466^8 / 8! = 5.2e-9).  About a third of the 64-bit operations of exp().
__device__ __forceinline__ double exp2_short(double y) {
  y = y < -1000.0 ? -1000.0 : y;
  const double n = floor(y + 0.5), r = (y - n) * 0.6931471805599453;
  double e = 1.0 / 5040;
  e = e * r + 1.0 / 720;
  e = e * r + 1.0 / 120;
  e = e * r + 1.0 / 24;
  e = e * r + 1.0 / 6;
  e = e * r + 0.5;
  e = e * r + 1.0;
  e = e * r + 1.0;
  return e * __longlong_as_double((long long)((int)n + 1023) << 52);
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

// A CTA per row.  The row's scores are kept in shared memory (kCached, up to
// kMostCached columns) or read again from memory for each pass; with the race
// they are overwritten by its values.
//
// A threshold ("the k-th largest", "the last one before the mass reaches p") is found
// with histograms over a linear map of the values, kBins bins from the largest to
// the smallest: counts, or exact masses as two 32-bit words (shared-memory atomics of 32 bits are
// native, and integer sums do not depend on their order).  The bin that holds the threshold is looked at
// again: its members are ranked against each other when there are at most
// kListed, else the map zooms into it.  Every zoom separates its largest from its smallest
// member, so it ends; members that are all equal are taken in index order.
//
// The race is run twice: in 32 bits over all kept candidates, as lower bounds
// with the arithmetic's error taken off, whose n-th largest leaves out everything
// that cannot be among the n best; and in 64 bits for the few that are left.
constexpr int kListed = 256;         // members that are ranked against each other
constexpr int kMostDrawn = 1024;     // draws of a row
constexpr int kRaced = 1536;         // candidates of a row that are raced in 64 bits
constexpr int kMostCached = 40960;   // columns of a row in shared memory

template <int THREADS>
struct Shared {
  static constexpr int kBins = 2 * THREADS;
  union {
    uint32_t bins[2][kBins];              // low and high words of a histogram
    struct {
      unsigned long long mass[kListed];   // of the ranked members, best first
      uint32_t key[kListed];
      int32_t index[kListed];
    } ranked;
    unsigned long long race[kRaced];      // order-preserving images of 64-bit race values
  };
  int32_t list[kRaced];
  unsigned long long words[2][THREADS / 32];
  unsigned long long found_above;
  uint32_t found_key;
  int32_t found_bin, found_index, members;
};

template <int THREADS>
struct Block {
  Shared<THREADS>& sh;
  int half = 0;

  // One barrier each: the next one uses the other words.
  template <typename V, typename Op>
  __device__ __forceinline__ V reduce(V v, Op op) {
    static_assert(sizeof(V) <= 8, "");
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
    V* words = reinterpret_cast<V*>(sh.words[half]);
    half ^= 1;
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = v;
    __syncthreads();
    v = words[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
    for (int off = THREADS / 64; off > 0; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
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
    unsigned long long* words = sh.words[half];
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

template <int THREADS, bool kCached>
__global__ void __launch_bounds__(THREADS) sample_rows_kernel(const __grid_constant__ Args A) {
  using S = Shared<THREADS>;
  constexpr int kBins = S::kBins;
  extern __shared__ float cache[];
  __shared__ S sh;
  Block<THREADS> block{sh};
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, C = A.cols, n = A.n;
  const float* const scores = A.scores + row * A.score_stride;
  const float* const uniforms = A.uniforms + row * A.uniform_stride;
  const double T = A.temperature.at(row);

  // the best candidate (key 0: there is none)
  uint32_t top = 0;
#pragma unroll 4
  for (int i = tid; i < C; i += THREADS) {
    const float v = scores[i];
    if (kCached) cache[i] = v;
    if (v > -INFINITY) top = max(top, key_of(v));
  }
  const uint32_t best_key = block.reduce(top, Most());  // and the barrier behind the cache
  int64_t* const indices = A.indices + row * n;
  float* const probabilities = A.probabilities + row * n;
  if (best_key == 0 || !(T > 0.0)) {
    for (int d = tid; d < n; d += THREADS) {
      indices[d] = -1;
      probabilities[d] = 0.f;
    }
    return;
  }
  const float best = value_of(best_key);
  const double best_d = best, inv_T = 1.0 / T;
  const float inv_Tf = (float)inv_T;
  const auto score = [&](int i) { return kCached ? cache[i] : scores[i]; };
  // the exponent, as defined; quickly and to within 1e-6 of its size; for masses
  const auto exponent = [&](float v) { return v == best ? 0.0 : ((double)v - best_d) / T; };
  const auto quick = [&](float v) { return v == best ? 0.f : fmaxf(v - best, -3.4e38f) * inv_Tf; };
  const double scale = ldexp(1.0, A.shift);
  const auto mass = [&](float v) {
    return __double2ull_rn(exp(v == best ? 0.0 : ((double)v - best_d) * inv_T) * scale);
  };
  const auto candidate = [&](float v) {  // false for NaN and -inf
    const float a = quick(v);
    return v > -INFINITY && (a > -699.f || (a > -701.f && exponent(v) >= kLeast));
  };

  // The filters keep a prefix: keys above `cut`, and those equal to it up to index `cut_index`.
  uint32_t cut = 0;
  int32_t cut_index = -1;
  const auto inside = [&](uint32_t key, int i) { return key > cut || (key == cut && i <= cut_index); };

  // Moves the cut.  The members are the candidates inside it whose weight is not
  // zero, of which `lowest` is the smallest key; weight(v) is what they add up, and
  // the new last member is the last one before which enough(sum) is false.
  const auto move_cut = [&](uint32_t lowest, auto weight, auto counts, auto enough, auto start) {
    constexpr bool kCounts = decltype(counts)::value;
    uint32_t high = best_key, low = lowest;
    unsigned long long above = 0;
    bool first = true;
    for (;;) {
      const float v_high = value_of(high);
      const float spread = v_high - value_of(low);
      const float per = spread < 3e38f ? (kBins - 1) / spread : 0.f;
      const auto bin_of = [&](float v) {  // falls with the value; in halves where a difference overflows
        const float t = per > 0.f ? (v_high - v) * per
                                  : (0.5f * v_high - 0.5f * v) * ((kBins - 1) / (0.5f * v_high - 0.5f * value_of(low)));
        return min((int)t, kBins - 1);
      };
      __syncthreads();  // whatever the words of the union held has been read
      for (int i = tid; i < kBins; i += THREADS) sh.bins[0][i] = sh.bins[1][i] = 0;
      if (tid == 0) sh.members = 0;
      __syncthreads();
      for (int i = tid; i < C; i += THREADS) {
        const float v = score(i);
        const uint32_t key = key_of(v);
        if (!candidate(v) || key < low || key > high || !inside(key, i)) continue;
        const int bin = low == high ? 0 : bin_of(v);
        if (kCounts) {
          // lanes of a warp that meet in one bin are added up first
          const unsigned active = __activemask();
          int same;
          __match_all_sync(active, bin, &same);
          if (!same) atomicAdd(&sh.bins[0][bin], 1u);
          else if ((tid & 31) == __ffs(active) - 1) atomicAdd(&sh.bins[0][bin], (uint32_t)__popc(active));
        } else {
          const unsigned long long w = weight(v);
          if (w) {
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&sh.bins[0][bin], lo);
            const uint32_t up = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
            if (up) atomicAdd(&sh.bins[1][bin], up);
          }
        }
      }
      __syncthreads();
      const int b0 = 2 * tid;
      const unsigned long long w0 = sh.bins[0][b0] + ((unsigned long long)sh.bins[1][b0] << 32);
      const unsigned long long w1 = sh.bins[0][b0 + 1] + ((unsigned long long)sh.bins[1][b0 + 1] << 32);
      unsigned long long total;
      const unsigned long long pre = above + block.before(w0 + w1, &total);
      if (first) start(total);  // the weight of all members: what enough() goes by
      first = false;
      if (!enough(pre) && enough(pre + w0)) {
        sh.found_bin = b0;
        sh.found_above = pre;
      } else if (!enough(pre + w0) && enough(pre + w0 + w1)) {
        sh.found_bin = b0 + 1;
        sh.found_above = pre + w0;
      }
      __syncthreads();
      const int bin = sh.found_bin;
      above = sh.found_above;
      uint32_t most = 0, least = 0xffffffffu;
      for (int i = tid; i < C; i += THREADS) {
        const float v = score(i);
        const uint32_t key = key_of(v);
        if (!candidate(v) || key < low || key > high || !inside(key, i)) continue;
        if ((low == high ? 0 : bin_of(v)) != bin) continue;
        most = max(most, key);
        least = min(least, key);
        const int at = atomicAdd(&sh.members, 1);
        if (at < kListed) sh.list[at] = i;
      }
      most = block.reduce(most, Most());
      least = block.reduce(least, Least());
      const int members = sh.members;
      if (members <= kListed) {
        uint32_t my_key = 0;
        int my_index = 0, rank = -1;
        if (tid < members) {
          my_index = sh.list[tid];
          my_key = key_of(score(my_index));
          sh.ranked.key[tid] = my_key;
        }
        static_assert(THREADS >= kListed, "a thread per ranked member");
        __syncthreads();
        if (tid < members) {
          rank = 0;
          for (int j = 0; j < members; ++j) {
            const uint32_t k = sh.ranked.key[j];
            rank += k > my_key || (k == my_key && sh.list[j] < my_index);
          }
        }
        __syncthreads();
        if (rank >= 0) {
          sh.ranked.key[rank] = my_key;
          sh.ranked.index[rank] = my_index;
          sh.ranked.mass[rank] = kCounts ? 1ull : weight(value_of(my_key));
        }
        __syncthreads();
        if (tid < 32) {  // the last member before which the sum is not enough
          unsigned long long sum = above;
          int last = 0;
          for (int base = 0; base < members; base += 32) {
            const unsigned long long w = base + tid < members ? sh.ranked.mass[base + tid] : 0;
            unsigned long long upto = w;
#pragma unroll
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
            sh.found_key = sh.ranked.key[last];
            sh.found_index = sh.ranked.index[last];
          }
        }
        __syncthreads();
        cut = sh.found_key;
        cut_index = sh.found_index;
        return;
      }
      if (most == least) {
        // More equal members than are listed: how many stay, and the index of the last of them.
        const unsigned long long each = kCounts ? 1ull : weight(value_of(most));
        int lo = 1, hi = members;  // the largest r with !enough(above + (r - 1) * each)
        while (lo < hi) {
          const int mid = lo + (hi - lo + 1) / 2;
          if (!enough(above + (unsigned long long)(mid - 1) * each)) lo = mid; else hi = mid - 1;
        }
        int from = 0, to = C - 1;  // the smallest index up to which there are lo of them
        while (from < to) {
          const int mid = from + (to - from) / 2;
          int some = 0;
          for (int i = tid; i <= mid; i += THREADS) {
            const float v = score(i);
            some += candidate(v) && key_of(v) == most && inside(most, i);
          }
          if (block.reduce(some, Add()) >= lo) to = mid; else from = mid + 1;
        }
        cut = most;
        cut_index = from;
        return;
      }
      high = most;
      low = least;
    }
  };

  const int64_t k = A.top_k.at(row);
  const double p = A.top_p.at(row);
  const bool by_mass = p > 0.0 && p < 1.0;
  if (k > 0 && k < C) {
    uint32_t least = 0xffffffffu;
    int some = 0;
    for (int i = tid; i < C; i += THREADS) {
      const float v = score(i);
      if (!candidate(v)) continue;
      least = min(least, key_of(v));
      ++some;
    }
    least = block.reduce(least, Least());
    some = block.reduce(some, Add());
    if (k < some) {
      const unsigned long long want = (unsigned long long)k;
      move_cut(least, [](float) { return 1ull; }, std::true_type(),
               [&](unsigned long long sum) { return sum >= want; }, [](unsigned long long) {});
    }
  }
  if (by_mass) {
    // the smallest member with a mass: below -(shift + 2) ln 2 a weight rounds to none
    const float none = -0.6931472f * (A.shift + 2);
    uint32_t least = 0xffffffffu;
    for (int i = tid; i < C; i += THREADS) {
      const float v = score(i);
      if (candidate(v) && quick(v) > none && inside(key_of(v), i)) least = min(least, key_of(v));
    }
    least = block.reduce(least, Least());
    double limit = 0.0;
    move_cut(least, mass, std::false_type(), [&](unsigned long long sum) { return !((double)sum < limit); },
             [&](unsigned long long total) { limit = p * (double)total; });
  }
  const double least_share = A.min_p.at(row);
  const bool by_share = least_share > 0.0 && least_share <= 1.0;
  const float share_exponent = by_share ? (float)log(least_share) : -INFINITY;
  const float share_margin = 1e-5f * (1.f - share_exponent);
  const auto kept = [&](float v, int i) {
    if (!candidate(v) || !inside(key_of(v), i)) return false;
    if (!by_share) return true;
    const float d = quick(v) - share_exponent;
    return d > share_margin || (d > -share_margin && exp(exponent(v)) >= least_share);
  };

  // The race in 32 bits: lower bounds.  a and the logarithms are off by at most a few
  // 2^-23 of their size, and the size of either is at most |sum| + 36 (a uniform
  // strictly between 0 and 1 has -4.7 < -log(-log u) < 16.7).
  const auto error_at = [](float g) { return 1e-6f * (fabsf(g) + 40.f); };
  const auto lower_race = [&](float v, float u) {
    const float g = quick(v) - logf(-logf(u));
    return g - error_at(g);
  };
  const bool exact_sum = k > 0 || by_mass;  // few are kept: the masses that the filters saw
  const double per_bit = inv_T * 1.4426950408889634;
  unsigned long long sum = 0;
  float g_most = -INFINITY, g_least = INFINITY;
  int open = 0, odd = 0;  // candidates in the race; uniforms of 0 and 1
  for (int i = tid; i < C; i += THREADS) {
    const float v = score(i);
    float g = -INFINITY;
    if (kept(v, i)) {
      sum += exact_sum ? mass(v) : v == best ? (unsigned long long)scale
                                             : __double2ull_rn(exp2_short(((double)v - best_d) * per_bit) * scale);
      const float u = uniforms[i];
      if (u > 0.f && u < 1.f) {
        g = lower_race(v, u);
        g_most = fmaxf(g_most, g);
        g_least = fminf(g_least, g);
        ++open;
      } else if (u == 0.f || u == 1.f) {
        odd |= u == 1.f ? 2 : 1;
      }
    }
    if (kCached) cache[i] = g;
  }
  const double total = (double)block.reduce(sum, Add());
  g_most = block.reduce(g_most, Most());
  g_least = block.reduce(g_least, Least());
  open = block.reduce(open, Add());
  odd = block.reduce(odd, [](int a, int b) { return a | b; });
  const auto race = [&](int i) {
    const float v = scores[i];
    const double r = exponent(v) - log(-log((double)uniforms[i]));
    return r < -1e300 ? -1e300 : r;  // a uniform of 0 comes last; NaN stays
  };
  const auto share = [&](int i) { return (float)(exp(exponent(scores[i])) * scale / total); };

  bool listed = !(odd & 2) && (open >= n || !(odd & 1));
  if (listed && open > 0) {
    const float g_spread = g_most - g_least;
    const float per = g_spread > 0.f ? (kBins - 1) / g_spread : 0.f;
    const auto bin_of = [&](float g) { return max(0, min((int)((g_most - g) * per), kBins - 1)); };
    const auto bound = [&](int i) {
      if (kCached) return cache[i];
      const float v = score(i), u = uniforms[i];
      return kept(v, i) && u > 0.f && u < 1.f ? lower_race(v, u) : -INFINITY;
    };
    __syncthreads();
    if (tid == 0) {
      sh.members = 0;
      sh.found_bin = kBins - 1;
    }
    if (open > n) {
      for (int i = tid; i < kBins; i += THREADS) sh.bins[0][i] = 0;
      __syncthreads();
      for (int i = tid; i < C; i += THREADS) {
        const float g = bound(i);
        if (g > -INFINITY) atomicAdd(&sh.bins[0][bin_of(g)], 1u);
      }
      __syncthreads();
      const unsigned long long c0 = sh.bins[0][2 * tid], c1 = sh.bins[0][2 * tid + 1];
      unsigned long long all;
      const unsigned long long pre = block.before(c0 + c1, &all), want = n;
      if (pre < want && pre + c0 >= want) sh.found_bin = 2 * tid;
      else if (pre + c0 < want && pre + c0 + c1 >= want) sh.found_bin = 2 * tid + 1;
    }
    __syncthreads();
    const int bin = sh.found_bin;
    for (int i = tid; i < C; i += THREADS) {
      const float g = bound(i);
      if (g > -INFINITY && bin_of(g + 2.01f * error_at(g)) <= bin) {
        const int at = atomicAdd(&sh.members, 1);
        if (at < kRaced) sh.list[at] = i;
      }
    }
    __syncthreads();
    const int members = sh.members;
    listed = members <= kRaced;
    if (listed) {
      for (int j = tid; j < members; j += THREADS) {
        const unsigned long long bits = (unsigned long long)__double_as_longlong(race(sh.list[j]) + 0.0);
        sh.race[j] = bits >> 63 ? ~bits : bits | (1ull << 63);
      }
      __syncthreads();
      for (int j = tid; j < members; j += THREADS) {
        const unsigned long long mine = sh.race[j];
        const int i = sh.list[j];
        int rank = 0;
        for (int o = 0; o < members; ++o) {
          const unsigned long long other = sh.race[o];
          rank += other > mine || (other == mine && sh.list[o] < i);
        }
        if (rank < n) {
          indices[rank] = i;
          probabilities[rank] = share(i);
        }
      }
      for (int d = members + tid; d < n; d += THREADS) {
        indices[d] = -1;
        probabilities[d] = 0.f;
      }
      return;
    }
  }
  // Uniforms of 0 or 1 among the draws, more equal race values than are
  // listed, or nobody in the race: one pass for each draw, over the row in memory.
  double last = INFINITY;
  int last_index = -1;
  bool more = true;
  for (int d = 0; d < n; ++d) {
    double g = -INFINITY;
    int at = C;
    if (more) {
      for (int i = tid; i < C; i += THREADS) {
        if (!kept(scores[i], i)) continue;
        const double r = race(i);
        if (!(r >= -1e300) || r > last || (r == last && i <= last_index)) continue;
        if (r > g) {
          g = r;
          at = i;
        }
      }
    }
    const double most = block.reduce(g, Most());
    const int first = block.reduce(g == most && most > -INFINITY ? at : C, Least());
    more = first < C;
    last = most;
    last_index = first;
    if (tid == 0) {
      indices[d] = more ? first : -1;
      probabilities[d] = more ? share(first) : 0.f;
    }
  }
}

}  // namespace sample
}  // namespace maxsim
