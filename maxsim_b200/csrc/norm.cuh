// Row normalisation on the way from an encoder into the scoring operators:
// layer norm and unit rows, forward and backward, over rows that lie
// [n_segments, L_max, dim] in memory.  With offsets, only a segment's first
// offsets[n+1] - offsets[n] rows count, and they are written back to back
// (the pack step of pack.cuh with the normalisation on the way).
//
//   layer norm   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r,
//                y = h w + b
//     backward   u = g w, dx = r (u - mean(u) - h mean(u h)), dw = sum g h, db = sum g
//   unit rows    m = max(|x|, eps), y = x / m
//     backward   |x| > eps: dx = (g - y (y . g)) / m, else dx = g / eps
//
// Everything between a load and the final rounding is 32-bit.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "async.cuh"

namespace maxsim {
namespace norm {

enum Kind : int { kLayer = 0, kUnit = 1 };

constexpr int kThreads = 256;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Which rows there are.  Token row j of segment n starts n * segment_stride + j *
// row_stride elements into the tokens; with offsets it counts for j < offsets[n+1] -
// offsets[n] and is row offsets[n] + j of the packed tensors, without them every row
// counts and is row n * L_max + j.
struct Rows {
  int64_t segment_stride, row_stride;  // in elements
  const int32_t* offsets;              // [n_segments + 1], or null
  int32_t n_segments, L_max;
  int32_t rows;   // packed rows: the ones at or beyond are never touched
  int32_t chunk;  // consecutive packed rows of a CTA
  int32_t dim;

  __device__ __forceinline__ int32_t start(int32_t n) const { return offsets ? offsets[n] : n * L_max; }
  // Where the last token row starts.
  __device__ __forceinline__ int64_t last() const {
    return (n_segments - 1) * segment_stride + (L_max - 1) * row_stride;
  }
  // Packed rows that belong to a segment.
  __device__ __forceinline__ int32_t used() const { return min(rows, start(n_segments)); }
};

// Walks the packed rows upwards and knows the segment it is in.  A warp looks its first segment up
// once (32 offsets at a time) and then only steps: no division and, within a
// segment, no load.  Offsets that are none (decreasing, longer than L_max) lead to a
// token row of the batch, never out of it.
struct Walker {
  int32_t n, first, end;  // segment n is packed rows [first, end)

  __device__ __forceinline__ void find(const Rows& t, int32_t row) {  // all lanes of a warp, same row
    if (!t.offsets) {
      n = min(row / t.L_max, t.n_segments - 1);
    } else {
      const int lane = threadIdx.x & 31;
      int32_t lo = 0, size = t.n_segments;
      while (size > 1) {  // the last segment that starts at or before the row lies in [lo, lo + size)
        const int32_t step = (size + 31) >> 5;
        const int32_t at = lane * step;
        const bool yes = at < size && t.offsets[lo + at] <= row;
        const int32_t k = max(__popc(__ballot_sync(0xffffffffu, yes)) - 1, 0) * step;
        lo += k;
        size = min(step, size - k);
      }
      n = lo;
    }
    first = t.start(n);
    end = t.start(n + 1);
  }
  __device__ __forceinline__ void seek(const Rows& t, int32_t row) {
    while (row >= end && n + 1 < t.n_segments) {
      ++n;
      first = end;
      end = t.start(n + 1);
    }
  }
  __device__ __forceinline__ int32_t token(const Rows& t, int32_t row) const {  // in the segment
    return (int32_t)min((uint32_t)(row - first), (uint32_t)(t.L_max - 1));
  }
  __device__ __forceinline__ int64_t from(const Rows& t, int32_t row) const {
    return n * t.segment_stride + token(t, row) * t.row_stride;
  }
  __device__ __forceinline__ int64_t slot(const Rows& t, int32_t row) const {
    return (int64_t)n * t.L_max + token(t, row);
  }
};

// E consecutive elements of a row, moved as one access (16, 4 or 2 bytes).
// Plain loads throughout: __ldg of a 16-bit element is an asm statement that the
// compiler may move in front of the test for a null pointer.
template <int BYTES> struct Word { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };
template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
  T v[E];
};
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> load_pack(const void* p) {
  using U = typename Word<sizeof(T) * E>::type;
  Pack<T, E> out;
  *reinterpret_cast<U*>(&out) = *reinterpret_cast<const U*>(p);
  return out;
}
template <typename T, int E>
__device__ __forceinline__ void store_pack(void* p, const Pack<T, E>& x) {
  using U = typename Word<sizeof(T) * E>::type;
  *reinterpret_cast<U*>(p) = *reinterpret_cast<const U*>(&x);
}

// The elements of a pack as floats: in pairs, on which one instruction works at a time
// (the kernels are short of instructions), or one by one.
struct Pair {
  unsigned long long bits;
};
__device__ __forceinline__ Pair pair_of(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.bits) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ float2 both_of(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.bits));
  return f;
}
__device__ __forceinline__ Pair add(Pair a, Pair b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.bits) : "l"(b.bits));
  return a;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.bits) : "l"(b.bits));
  return a;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(a.bits) : "l"(b.bits), "l"(c.bits));
  return a;
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float total(Pair p) { const float2 f = both_of(p); return f.x + f.y; }
__device__ __forceinline__ float total(float f) { return f; }
__device__ __forceinline__ float most(Pair p) { const float2 f = both_of(p); return fmaxf(fabsf(f.x), fabsf(f.y)); }
__device__ __forceinline__ float most(float f) { return fabsf(f); }
template <typename X> __device__ __forceinline__ X splat(float f);
template <> __device__ __forceinline__ Pair splat<Pair>(float f) { return pair_of(f, f); }
template <> __device__ __forceinline__ float splat<float>(float f) { return f; }

template <int E>
using Elem = typename std::conditional<E % 2 == 0, Pair, float>::type;
template <int E>
constexpr int kElems = E % 2 == 0 ? E / 2 : 1;

template <typename T, int E>
__device__ __forceinline__ void expand(const Pack<T, E>& p, Elem<E> (&f)[kElems<E>]) {
  if constexpr (E % 2 != 0) {
    f[0] = widen(p.v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = pair_of(p.v[2 * i], p.v[2 * i + 1]);
      } else {
        const uint32_t u = reinterpret_cast<const uint32_t*>(&p)[i];
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of a float
          f[i] = pair_of(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
        } else {
          const float2 both = __half22float2(reinterpret_cast<const __half2&>(u));
          f[i] = pair_of(both.x, both.y);
        }
      }
    }
  }
}
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> compress(const Elem<E> (&f)[kElems<E>]) {
  Pack<T, E> p;
  if constexpr (E % 2 != 0) {
    p.v[0] = narrow<T>(f[0]);
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 both = both_of(f[i]);
      if constexpr (sizeof(T) == 4) {
        p.v[2 * i] = both.x;
        p.v[2 * i + 1] = both.y;
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        reinterpret_cast<__nv_bfloat162*>(&p)[i] = __floats2bfloat162_rn(both.x, both.y);
      } else {
        reinterpret_cast<__half2*>(&p)[i] = __floats2half2_rn(both.x, both.y);
      }
    }
  }
  return p;
}

template <int E>
__device__ __forceinline__ Pack<float, E> unpacked(const Elem<E> (&f)[kElems<E>]) {
  return compress<float, E>(f);
}

// A layer norm's weight or bias: float, or of the rows' type.
struct Affine {
  const void* p;  // null: none
  bool f32;
  // Elements c .. c + E - 1, where p and c are on multiples of the rows' packs.
  template <typename T, int E, bool F32>
  __device__ __forceinline__ void pack_as(int c, Elem<E> (&w)[kElems<E>]) const {
    const float* const floats = static_cast<const float*>(p) + c;
    if constexpr (!F32) {
      expand(load_pack<T, E>(static_cast<const T*>(p) + c), w);
    } else if constexpr (E % 4 == 0) {
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        const Pack<float, 4> f = load_pack<float, 4>(floats + 4 * i);
        w[2 * i] = pair_of(f.v[0], f.v[1]);
        w[2 * i + 1] = pair_of(f.v[2], f.v[3]);
      }
    } else if constexpr (E == 2) {
      w[0] = pair_of(floats[0], floats[1]);
    } else {
      w[0] = floats[0];
    }
  }
  template <typename T, int E>
  __device__ __forceinline__ void pack(int c, Elem<E> (&w)[kElems<E>]) const {
    if (f32) pack_as<T, E, true>(c, w);
    else pack_as<T, E, false>(c, w);
  }
};

// A vector of the row's width in shared memory, as floats.  A thread's pack of
// eight lies in two halves, so that neighbouring packs of a half meet no bank twice.
template <int E>
struct Wide {
  static constexpr int kPart = E < 4 ? E : 4;
  float* words;
  int packs;  // of the row
  static constexpr __host__ __device__ int bytes(int dim) { return (dim + E - 1) / E * E * 4; }
  template <typename T>
  __device__ __forceinline__ void fill(const Affine& a, int dim, float none) const {
    if (a.f32) put<T, true>(a, dim, none);
    else put<T, false>(a, dim, none);
  }
  // Several packs in flight (32 bf16 rows of 4096, whole kernel: 3.5 us; one element after the other 11.5).
  template <typename T, bool F32>
  __device__ __forceinline__ void put(const Affine& a, int dim, float none) const {
    constexpr int kAtOnce = E == 1 ? 8 : 4;
    for (int first = threadIdx.x; first < packs; first += kAtOnce * blockDim.x) {
      Elem<E> f[kAtOnce][kElems<E>];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int pack = first + i * blockDim.x;
        if (a.p && pack < packs) {
          a.pack_as<T, E, F32>(pack * E, f[i]);
        } else {
#pragma unroll
          for (int k = 0; k < kElems<E>; ++k) f[i][k] = splat<Elem<E>>(none);
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int pack = first + i * blockDim.x;
        if (pack >= packs) break;
        const Pack<float, E> w = unpacked<E>(f[i]);
#pragma unroll
        for (int k = 0; k < E / kPart; ++k)
          store_pack<float, kPart>(words + (k * packs + pack) * kPart,
                                   reinterpret_cast<const Pack<float, kPart>*>(&w)[k]);
      }
    }
  }
  __device__ __forceinline__ void get(int pack, Elem<E> (&w)[kElems<E>]) const {
#pragma unroll
    for (int i = 0; i < E / kPart; ++i) {
      const Pack<float, kPart> f = load_pack<float, kPart>(words + (i * packs + pack) * kPart);
      if constexpr (E % 2 != 0) {
        w[0] = f.v[0];
      } else {
#pragma unroll
        for (int e = 0; e < kPart / 2; ++e) w[i * kPart / 2 + e] = pair_of(f.v[2 * e], f.v[2 * e + 1]);
      }
    }
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// The factors of a unit row.  Nearly every row is plain: its sum of squares is well inside
// the 32-bit range and above eps^2, and y = x * rsqrt(sum).  For the others the sum is
// taken again over x / top, top = max|x|: y = (x / top) * inv.
struct UnitScale {
  float inv;
  bool scaled;   // inv belongs to x / top, else to x
  bool clamped;  // |x| <= eps: y = x / eps
};
__device__ __forceinline__ float least_square(float eps) { return fmaxf(1e-30f, 1.0001f * eps * eps); }
__device__ __forceinline__ bool plain_square(float ss, float least) { return ss > least && ss < 1e37f; }
// 1 / top as a product of two factors that both lie in the range, a power of two first.
__device__ __forceinline__ float2 reciprocal_parts(float top) {
  const float power = top > 1.f ? 5.421010862427522e-20f : 1.8446744073709552e19f;  // 2^-64, 2^64
  return make_float2(power, 1.0f / (top * power));
}
// `ss` is that of x / top where top is positive and finite, else of x; a NaN stays one.
__device__ __forceinline__ UnitScale unit_scale(float ss, float top, float eps) {
  const bool scaled = top > 0.f && top < INFINITY;
  const float norm = scaled ? top * sqrtf(ss) : sqrtf(ss);
  UnitScale u;
  if (norm == INFINITY && !scaled) {  // an infinity in the row: finite / inf = 0, inf / inf = NaN
    u.inv = 0.0f;
    u.scaled = u.clamped = false;
    return u;
  }
  u.clamped = norm <= eps;
  u.scaled = scaled && !u.clamped;
  u.inv = u.clamped ? 1.0f / eps : 1.0f / sqrtf(ss);
  return u;
}

// ---------------------------------------------------------------------------
// Rows shared by a team of TEAM threads (2 to 32 lanes of a warp, or a CTA of
// 128); a thread has V packs of E elements of a row.  Every element is read once and
// written once.
//
// HBM-bound for rows of wide packs: 5.3 to 6.2 TB/s of a copy's 6.5.  Every thread copies its own packs
// of the next row into a ring in shared memory (cp.async) and reads back nothing but
// what it copied itself, so the ring needs no barrier (odd rows of 16-bit elements are read back by other lanes of
// the warp and take a __syncwarp on either side); the reductions and the store of a row run under the loads of the
// next.
// ---------------------------------------------------------------------------
constexpr int kWide = 128;  // threads of a team that is a CTA

template <int TEAM>
constexpr int kCtaThreads = TEAM > 32 ? TEAM : kThreads;

// Threads an SM is to hold at once: what the registers are cut to.  More threads are more
// rows in flight, which past some point only hold the stores up.  Measured, 10^8 elements, us: layer norm
// forward, 98k x 1024 bf16, 256 / 512 / 768 threads: 91 / 69 / 80; 781k x 128, 512 / 768 / 1024: 79 / 69 / 80; teams of a
// CTA with four packs, which wait at barriers, 24k x 4096, 512 / 768: 110 / 103, before the weights were staged in
// packs (79 with 768 since).  Shared memory, which holds the weights as floats, has room for fewer of these than the
// registers (five of six at 2304, three at 4096), and rows are split evenly over all that are launched: 48k x 2048
// take 71, 43k x 2304 113.  Rows without wide packs are short of instructions instead and take all they get.  Layer norm backward, 781k x 128 and 300k x 333 bf16, 512 / 768: 128 / 117
// and 293 / 258; unit rows backward, 391k x 384 bf16, 256 / 512 / 768: 108 / 103 / 115.
template <int E, int TEAM, int V>
constexpr int kForwardThreads = V * E <= 8                               ? 1024
                                : E < 4                                  ? (V * E <= 16 ? 1024 : 768)
                                : V * E <= 16                            ? 768
                                : E == 8 && TEAM == kWide                ? 768
                                                                         : 512;
template <int KIND, int E, int TEAM, int V>
constexpr int kBackwardThreads = KIND == kUnit ? (V * E <= 8 ? 1024 : V * E <= 16 ? 768 : 512)
                                 : V * E <= 8 || (V * E <= 16 && TEAM <= 32) ? 768
                                                                             : 512;
// CTAs of a layer norm's backward kernel that an SM is to hold at most, whatever the instantiation (six of 128
// threads; the host asserts it): each writes one row of partial sums, and the workspace has room for as many.
constexpr int kSumCtas = 6;

// How a row's elements get into the ring: a thread's own packs of 16 or 4 bytes; for rows of
// 16-bit elements that start and end anywhere, the 4-byte words around them, which
// the lanes of a warp read from each other; or not at all (such rows shared by a CTA).
enum Staging : int { kInPlace = 0, kPacks = 1, kWords = 2 };
template <typename T, int E, int TEAM>
constexpr Staging kStaging = sizeof(T) * E >= 4 ? kPacks : TEAM == 32 ? kWords : kInPlace;

// Rows in the ring, one of them in use.  More loads in flight did not help, they held the
// stores up: 2, 3 and 4 stages took 159, 174 and 176 us for 2.4M x 96 fp16 unit rows (backward 222, 248, 249),
// 69, 78 and 75 for a layer norm of 98k x 1024 bf16 rows.  A CTA that takes a row together, with barriers
// between, is short of them forward: 199 us with 2, 156 with 3 or 4, for 24k x 4096 fp32 rows.
template <int TEAM, int TENSORS>
constexpr int kStages = TEAM > 32 && TENSORS == 1 ? 3 : 2;
// Bytes of one tensor's part of a stage, all threads of the CTA.
template <typename T, int E, int TEAM, int V>
constexpr int kPartBytes = kStaging<T, E, TEAM> == kWords ? kCtaThreads<TEAM> / 32 * (64 * V + 16)
                                                          : kCtaThreads<TEAM> * V * E * (int)sizeof(T);
template <typename T, int E, int TEAM, int V, int TENSORS>
constexpr int kRingBytes = kStaging<T, E, TEAM> == kInPlace
                               ? 0
                               : kStages<TEAM, TENSORS> * TENSORS * kPartBytes<T, E, TEAM, V>;

// The column sums at the end of the backward kernel take the ring's place: element e
// of a pack lies e * kSumPitch on, which meets no bank twice, written or read.
template <int E, int TEAM>
constexpr int kSumPitch = TEAM + 32 / E;
template <int E, int TEAM>
constexpr int kSumBytes = 2 * (kCtaThreads<TEAM> / TEAM) * E * kSumPitch<E, TEAM> * 4;

// What lies before the weights in the backward kernel's shared memory.
template <typename T, int KIND, int E, int TEAM, int V>
constexpr int kBackwardBytes = [] {
  const int ring = kRingBytes<T, E, TEAM, V, 2>;
  const int sums = KIND == kLayer ? kSumBytes<E, TEAM> : 0;
  return ring > sums ? ring : sums;
}();

// Sums over a team.  Teams of one warp or less use shuffles: all lanes of the
// warp take part, whether their row counts or not.  A CTA team takes one
// barrier per sum: the next sum uses the other half of the words.
template <int TEAM>
struct Team {
  float* words;  // [2][2][TEAM / 32] for a CTA
  int half = 0;
  __device__ __forceinline__ Team(float* w) : words(w) {}

  template <typename Op>
  __device__ __forceinline__ float2 reduce(float a, float b, Op op) {
#pragma unroll
    for (int off = (TEAM > 32 ? 32 : TEAM) / 2; off > 0; off >>= 1) {
      a = op(a, __shfl_xor_sync(0xffffffffu, a, off));
      b = op(b, __shfl_xor_sync(0xffffffffu, b, off));
    }
    if constexpr (TEAM > 32) {
      constexpr int W = TEAM / 32;
      float* mine = words + half * 2 * W;
      half ^= 1;
      if ((threadIdx.x & 31) == 0) {
        mine[threadIdx.x >> 5] = a;
        mine[W + (threadIdx.x >> 5)] = b;
      }
      __syncthreads();
      a = mine[0];
      b = mine[W];
#pragma unroll
      for (int w = 1; w < W; ++w) {
        a = op(a, mine[w]);
        b = op(b, mine[W + w]);
      }
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float2 sums(float a, float b) {
    return reduce(a, b, [](float x, float y) { return x + y; });
  }
  // The second value is unused and goes with the optimiser (for a CTA it costs a word).
  __device__ __forceinline__ float sum(float a) { return sums(a, 0.f).x; }
  __device__ __forceinline__ float max(float a) {
    return reduce(a, 0.f, [](float x, float y) { return fmaxf(x, y); }).x;
  }
  // Whether any team that has to run the same shuffles says yes.
  __device__ __forceinline__ bool any(bool v) const {
    return TEAM > 32 ? v : (bool)__any_sync(0xffffffffu, v);
  }
};

// The rows ahead, of TENSORS tensors.
template <typename T, int E, int TEAM, int V, int TENSORS>
struct Ring {
  static constexpr Staging kHow = kStaging<T, E, TEAM>;
  static constexpr int kBytes = E * (int)sizeof(T);
  static constexpr int kCta = kCtaThreads<TEAM>;
  static constexpr int kPart = kPartBytes<T, E, TEAM, V>;
  char* mine;
  int lane;
  __device__ __forceinline__ Ring(char* shared)
      : mine(shared + (kHow == kWords ? (threadIdx.x >> 5) * (64 * V + 16) : threadIdx.x * kBytes)),
        lane(threadIdx.x % TEAM) {}
  __device__ __forceinline__ char* at(int stage, int tensor) const {
    return mine + (stage * TENSORS + tensor) * kPart;
  }
  // Before a stage is filled again: in kWords other lanes have read it.
  __device__ __forceinline__ void reuse() const {
    if (kHow == kWords) __syncwarp();
  }
  __device__ __forceinline__ void filled() const {
    if (kHow == kWords) __syncwarp();
  }
  // `edge`: the row is the first or last of the tensor, whose outer words are not whole.
  __device__ __forceinline__ void copy(int stage, int tensor, const T* row, int dim, bool edge) const {
    if constexpr (kHow == kWords) {
      const int odd = (int)((uintptr_t)row >> 1) & 1, elements = dim + odd, words = (elements + 1) >> 1;
      const T* from = row - odd;
      char* to = at(stage, tensor);
#pragma unroll
      for (int v = 0; v <= V / 2; ++v) {
        const int k = lane + 32 * v;
        if (k >= words) break;
        const bool torn = edge && ((k == 0 && odd) || (k == words - 1 && (elements & 1)));
        if (!torn) {
          copy_async<4>(to + 4 * k, from + 2 * k);
        } else {
          if (k > 0 || !odd) reinterpret_cast<T*>(to)[2 * k] = from[2 * k];
          if (2 * k + 1 < elements) reinterpret_cast<T*>(to)[2 * k + 1] = from[2 * k + 1];
        }
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (lane + TEAM * v) * E;
        if (c < dim) copy_async<kBytes>(at(stage, tensor) + v * (kCta * kBytes), row + c);
      }
    }
  }
  // Pack v of this thread; `row` is where the row was copied from.
  __device__ __forceinline__ Pack<T, E> pack(int stage, int tensor, int v, const T* row) const {
    if constexpr (kHow == kWords) {
      const int odd = (int)((uintptr_t)row >> 1) & 1;
      return load_pack<T, E>(reinterpret_cast<const T*>(at(stage, tensor)) + odd + lane + 32 * v);
    } else {
      return load_pack<T, E>(at(stage, tensor) + v * (kCta * kBytes));
    }
  }
};

// The packed rows of a CTA: t.chunk consecutive ones, which its teams take in turn, so that
// what a CTA reads and writes at any moment lies together (295k x 768 bf16 rows packed out of 1024 x 512, backward:
// 309 us; with consecutive rows for every warp 323 us).
template <int TEAM>
struct Turn {
  static constexpr int kRows = kCtaThreads<TEAM> / TEAM;  // rows at a time
  int32_t begin, end, mine;  // of the CTA; the team's place in its turn
  __device__ __forceinline__ Turn(const Rows& t) {
    const int64_t from = (int64_t)blockIdx.x * t.chunk, used = t.used();
    begin = (int32_t)min(from, used);
    end = (int32_t)min(from + t.chunk, used);
    mine = threadIdx.x / TEAM;
  }
};

template <typename T, int KIND, int E, int TEAM, int V>
__global__ void __launch_bounds__(kCtaThreads<TEAM>, kForwardThreads<E, TEAM, V> / kCtaThreads<TEAM>)
forward_rows_kernel(const T* __restrict__ tokens, const __grid_constant__ Rows t, Affine weight, Affine bias,
                    T* __restrict__ out, float* __restrict__ mean, float* __restrict__ rstd, float eps) {
  constexpr Staging kHow = kStaging<T, E, TEAM>;
  constexpr int S = kHow != kInPlace ? kStages<TEAM, 1> : 1;
  extern __shared__ __align__(16) char shared[];
  __shared__ float words[TEAM > 32 ? TEAM / 8 : 1];
  Team<TEAM> team(words);
  const Ring<T, E, TEAM, V, 1> ring(shared);
  const int lane = threadIdx.x % TEAM;
  const float per = 1.0f / t.dim, least = least_square(eps);
  const Turn<TEAM> turn(t);
  constexpr int R = Turn<TEAM>::kRows;

  Walker ahead, here;
  if (turn.begin < turn.end) ahead.find(t, turn.begin);
  here = ahead;
  const auto copy = [&](int stage, int32_t row) {
    if (row < turn.end) {
      ahead.seek(t, row);
      const int64_t from = ahead.from(t, row);
      ring.copy(stage, 0, tokens + from, t.dim, from == 0 || from == t.last());
    }
    copies_commit();
  };
  if constexpr (kHow != kInPlace) {
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy(i, turn.begin + turn.mine + i * R);
  }
  const int packs = (t.dim + E - 1) / E;
  float* const after = reinterpret_cast<float*>(shared + kRingBytes<T, E, TEAM, V, 1>);
  const Wide<E> w{after, packs}, b{after + packs * E, packs};
  if constexpr (KIND == kLayer) {
    w.template fill<T>(weight, t.dim, 1.0f);
    b.template fill<T>(bias, t.dim, 0.0f);
    __syncthreads();
  }
  int stage = 0;
  for (int32_t at = turn.begin; at < turn.end; at += R) {
    const int32_t row = at + turn.mine;
    const bool there = row < turn.end;
    if constexpr (kHow != kInPlace) {
      ring.reuse();
      copy(stage == 0 ? S - 1 : stage - 1, row + (S - 1) * R);
      copies_wait<S - 1>();
      ring.filled();
    }
    const T* x = tokens;
    if (kHow != kPacks && there) {
      here.seek(t, row);
      x += here.from(t, row);
    }
    using X = Elem<E>;
    constexpr int N = kElems<E>;
    X f[V][N];  // zero where there is no element
    X sum = splat<X>(0.f);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (lane + TEAM * v) * E;
      if (there && c < t.dim) {
        if constexpr (kHow != kInPlace) expand(ring.pack(stage, 0, v, x), f[v]);
        else expand(load_pack<T, E>(x + c), f[v]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[v][i] = splat<X>(0.f);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) sum = KIND == kLayer ? add(f[v][i], sum) : fma(f[v][i], f[v][i], sum);
    }
    stage = stage == S - 1 ? 0 : stage + 1;
    if constexpr (KIND == kLayer) {
      const float mu = team.sum(total(sum)) * per;
      const X minus_mu = splat<X>(-mu);
      sum = splat<X>(0.f);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if ((lane + TEAM * v) * E < t.dim) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            f[v][i] = add(f[v][i], minus_mu);
            sum = fma(f[v][i], f[v][i], sum);
          }
        }
      }
      const float r = rsqrtf(team.sum(total(sum)) * per + eps);
      if (there) {
        T* const y = out + (int64_t)row * t.dim;
        const X rr = splat<X>(r);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int c = (lane + TEAM * v) * E;
          if (c < t.dim) {
            X wv[N], bv[N];
            w.get(lane + TEAM * v, wv);
            b.get(lane + TEAM * v, bv);
#pragma unroll
            for (int i = 0; i < N; ++i) f[v][i] = fma(mul(f[v][i], rr), wv[i], bv[i]);
            store_pack<T, E>(y + c, compress<T, E>(f[v]));
          }
        }
        if (mean && lane == 0) {
          mean[row] = mu;
          rstd[row] = r;
        }
      }
    } else {
      const float ss = team.sum(total(sum));
      float inv = rsqrtf(ss);
      const bool plain = plain_square(ss, least) || !there;
      if (team.any(!plain)) {
        float top = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int i = 0; i < N; ++i) top = fmaxf(top, most(f[v][i]));
        top = team.max(top);
        const bool scaled = top > 0.f && top < INFINITY;
        // x / top by its reciprocal, in two factors that do not leave the range
        const float2 by = scaled ? reciprocal_parts(top) : make_float2(1.f, 1.f);
        X again = splat<X>(0.f);
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const X d = mul(mul(f[v][i], splat<X>(by.x)), splat<X>(by.y));
            again = fma(d, d, again);
          }
        const float ss2 = team.sum(total(again));
        if (!plain) {
          const UnitScale u = unit_scale(scaled ? ss2 : ss, top, eps);
          inv = u.inv;
          if (u.scaled) {
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
              for (int i = 0; i < N; ++i) f[v][i] = mul(mul(f[v][i], splat<X>(by.x)), splat<X>(by.y));
          }
        }
      }
      if (there) {
        T* const y = out + (int64_t)row * t.dim;
        const X ii = splat<X>(inv);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int c = (lane + TEAM * v) * E;
          if (c < t.dim) {
#pragma unroll
            for (int i = 0; i < N; ++i) f[v][i] = mul(f[v][i], ii);
            store_pack<T, E>(y + c, compress<T, E>(f[v]));
          }
        }
      }
    }
  }
}

// Zeroes the token rows that do not count, in grad_tokens: the units share the
// slots, and what is not valid of a segment lies in one piece.
template <typename T, int E>
__device__ __forceinline__ void zero_padding(const Rows& t, T* grad_tokens, int64_t unit, int64_t units, int lane, int team) {
  const int64_t slots = (int64_t)t.n_segments * t.L_max, share = (slots + units - 1) / units;
  const int64_t lo = unit * share, hi = min(lo + share, slots);
  const int32_t used = t.used();
  Pack<T, E> zero;
#pragma unroll
  for (int e = 0; e < E; ++e) zero.v[e] = narrow<T>(0.f);
  for (int64_t n = lo / t.L_max; n * t.L_max < hi; ++n) {
    const int32_t first = t.offsets[n];
    const int32_t len = max(min(min(t.offsets[n + 1], used) - first, t.L_max), 0);
    const int64_t from = max(lo, n * t.L_max + len) * t.dim, to = min(hi, (n + 1) * t.L_max) * t.dim;
    for (int64_t c = from + lane * E; c < to; c += team * E) store_pack<T, E>(grad_tokens + c, zero);
  }
}

// The gradient of the rows and, for a layer norm, a CTA's share of the weight's
// and bias's: a thread meets the same columns in every row, so it sums
// g h and g in registers over all its rows; at the end the teams of the CTA add up
// through shared memory and the CTA writes one row of partial [2][gridDim.x][dim].
// The row's packs are read twice from the ring (once for the sums, once for the result):
// the registers go to the column sums.
template <typename T, int KIND, int E, int TEAM, int V>
__global__ void __launch_bounds__(kCtaThreads<TEAM>, kBackwardThreads<KIND, E, TEAM, V> / kCtaThreads<TEAM>)
backward_rows_kernel(const T* __restrict__ grad, const T* __restrict__ tokens, const __grid_constant__ Rows t,
                     Affine weight, const float* __restrict__ mean, const float* __restrict__ rstd,
                     T* __restrict__ grad_tokens, float* __restrict__ partial, float eps) {
  constexpr int kCta = kCtaThreads<TEAM>;
  constexpr Staging kHow = kStaging<T, E, TEAM>;
  constexpr int S = kHow != kInPlace ? kStages<TEAM, 2> : 1;
  constexpr int kFixed = kBackwardBytes<T, KIND, E, TEAM, V>;
  extern __shared__ __align__(16) char shared[];
  __shared__ float words[TEAM > 32 ? TEAM / 8 : 1];
  Team<TEAM> team(words);
  const Ring<T, E, TEAM, V, 2> ring(shared);
  const int lane = threadIdx.x % TEAM;
  const float per = 1.0f / t.dim, least = least_square(eps);
  Elem<E> dw[KIND == kLayer ? V : 1][kElems<E>], db[KIND == kLayer ? V : 1][kElems<E>];
  if constexpr (KIND == kLayer) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < kElems<E>; ++i) dw[v][i] = db[v][i] = splat<Elem<E>>(0.f);
  }
  const Turn<TEAM> turn(t);
  constexpr int R = Turn<TEAM>::kRows;
  Walker ahead, here;
  if (turn.begin < turn.end) ahead.find(t, turn.begin);
  here = ahead;
  const auto copy = [&](int stage, int32_t row) {
    if (row < turn.end) {
      ahead.seek(t, row);
      const int64_t from = ahead.from(t, row);
      ring.copy(stage, 0, tokens + from, t.dim, from == 0 || from == t.last());
      ring.copy(stage, 1, grad + (int64_t)row * t.dim, t.dim, row == 0 || row == t.rows - 1);
    }
    copies_commit();
  };
  if constexpr (kHow != kInPlace) {
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy(i, turn.begin + turn.mine + i * R);
  }
  const int packs = (t.dim + E - 1) / E;
  const Wide<E> w{reinterpret_cast<float*>(shared + kFixed), packs};
  if constexpr (KIND == kLayer) {
    w.template fill<T>(weight, t.dim, 1.0f);
    __syncthreads();
  }
  if (t.offsets && grad_tokens) {
    if (TEAM > 32) zero_padding<T, E>(t, grad_tokens, blockIdx.x, gridDim.x, threadIdx.x, TEAM);
    else zero_padding<T, E>(t, grad_tokens, (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5),
                            (int64_t)gridDim.x * (kThreads / 32), threadIdx.x & 31, 32);
  }
  int stage = 0;
  for (int32_t at = turn.begin; at < turn.end; at += R) {
    const int32_t row = at + turn.mine;
    const bool there = row < turn.end;
    float mu = 0.f, r = 0.f;
    if (there) {
      here.seek(t, row);
      if (KIND == kLayer) {
        mu = mean[row];
        r = rstd[row];
      }
    }
    if constexpr (kHow != kInPlace) {
      ring.reuse();
      copy(stage == 0 ? S - 1 : stage - 1, row + (S - 1) * R);
      copies_wait<S - 1>();
      ring.filled();
    }
    const T* const x_row = tokens + (kHow != kPacks && there ? here.from(t, row) : 0);
    const T* const g_row = grad + (there ? (int64_t)row * t.dim : 0);
    using X = Elem<E>;
    constexpr int N = kElems<E>;
    // pack v of the row and of its gradient
    const auto packs_of = [&](int v, X (&x)[N], X (&g)[N]) {
      if constexpr (kHow != kInPlace) {
        expand(ring.pack(stage, 0, v, x_row), x);
        expand(ring.pack(stage, 1, v, g_row), g);
      } else {
        const int c = (lane + TEAM * v) * E;
        expand(load_pack<T, E>(x_row + c), x);
        expand(load_pack<T, E>(g_row + c), g);
      }
    };
    T* const dx = grad_tokens + (there ? here.slot(t, row) * t.dim : 0);
    const bool store = grad_tokens && there;
    if constexpr (KIND == kLayer) {
      X su = splat<X>(0.f), suh = su;
      const X minus_mu = splat<X>(-mu), rr = splat<X>(r);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (there && (lane + TEAM * v) * E < t.dim) {
          X x[N], g[N], wv[N];
          packs_of(v, x, g);
          w.get(lane + TEAM * v, wv);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const X h = mul(add(x[i], minus_mu), rr), u = mul(g[i], wv[i]);
            su = add(u, su);
            suh = fma(u, h, suh);
            dw[v][i] = fma(g[i], h, dw[v][i]);
            db[v][i] = add(g[i], db[v][i]);
          }
        }
      }
      const float2 both = team.sums(total(su), total(suh));
      // dx = r (u - mean(u) - h mean(u h))
      const X minus_u = splat<X>(-r * (both.x * per)), minus_h = splat<X>(-r * (both.y * per));
      asm volatile("" ::: "memory");  // read the packs again instead of keeping them
      if (store) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int c = (lane + TEAM * v) * E;
          if (c < t.dim) {
            X x[N], g[N], wv[N];
            packs_of(v, x, g);
            w.get(lane + TEAM * v, wv);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const X h = mul(add(x[i], minus_mu), rr);
              x[i] = fma(mul(g[i], wv[i]), rr, fma(h, minus_h, minus_u));
            }
            store_pack<T, E>(dx + c, compress<T, E>(x));
          }
        }
      }
    } else {
      X x[V][N], g[V][N];
      X squares = splat<X>(0.f), products = squares;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (there && (lane + TEAM * v) * E < t.dim) {
          packs_of(v, x[v], g[v]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) x[v][i] = g[v][i] = splat<X>(0.f);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          squares = fma(x[v][i], x[v][i], squares);
          products = fma(x[v][i], g[v][i], products);
        }
      }
      const float2 both = team.sums(total(squares), total(products));
      const float ss = both.x, xg = both.y;
      float inv = rsqrtf(ss), scale = inv, along = xg * inv;  // along: y . g; dx = (g - y along) * scale
      const bool plain = plain_square(ss, least) || !there;
      if (team.any(!plain)) {
        float top = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int i = 0; i < N; ++i) top = fmaxf(top, most(x[v][i]));
        top = team.max(top);
        const bool scaled = top > 0.f && top < INFINITY;
        const float2 by = scaled ? reciprocal_parts(top) : make_float2(1.f, 1.f);
        squares = products = splat<X>(0.f);
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const X d = mul(mul(x[v][i], splat<X>(by.x)), splat<X>(by.y));
            squares = fma(d, d, squares);
            products = fma(d, g[v][i], products);
          }
        const float2 again = team.sums(total(squares), total(products));
        if (!plain) {
          const UnitScale u = unit_scale(scaled ? again.x : ss, top, eps);
          inv = scale = u.inv;
          along = u.clamped ? 0.0f : (scaled ? again.y : xg) * inv;
          if (u.scaled) {
            scale = inv * by.x * by.y;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
              for (int i = 0; i < N; ++i) x[v][i] = mul(mul(x[v][i], splat<X>(by.x)), splat<X>(by.y));
          }
        }
      }
      if (store) {
        const X ii = splat<X>(inv), kk = splat<X>(scale), minus = splat<X>(-along);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int c = (lane + TEAM * v) * E;
          if (c < t.dim) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[v][i] = mul(fma(mul(x[v][i], ii), minus, g[v][i]), kk);
            store_pack<T, E>(dx + c, compress<T, E>(x[v]));
          }
        }
      }
    }
    stage = stage == S - 1 ? 0 : stage + 1;
  }
  if constexpr (KIND == kLayer) {
    if (!partial) return;
    constexpr int kTeams = kCta / TEAM, kPitch = kSumPitch<E, TEAM>;
    float(*acc)[kTeams][E * kPitch] = reinterpret_cast<float(*)[kTeams][E * kPitch]>(shared);
    copies_wait<0>();  // every copy was waited for where its row was used; the ring is free
#pragma unroll
    for (int v = 0; v < V; ++v) {
      __syncthreads();
      const Pack<float, E> pw = unpacked<E>(dw[v]), pb = unpacked<E>(db[v]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        acc[0][threadIdx.x / TEAM][e * kPitch + lane] = pw.v[e];
        acc[1][threadIdx.x / TEAM][e * kPitch + lane] = pb.v[e];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * TEAM * E; i += kCta) {
        const int which = i / (TEAM * E), c = i % (TEAM * E);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kTeams; ++k) sum += acc[which][k][(c % E) * kPitch + c / E];
        const int col = TEAM * E * v + c;
        if (col < t.dim) partial[((int64_t)which * gridDim.x + blockIdx.x) * t.dim + col] = sum;
      }
    }
  }
}

// Adds the rows of partial [2][slabs][dim] in a fixed order: a CTA takes 32 columns of
// one of the two halves, its 32 warps every 32nd row.
constexpr int kSumThreads = 1024;
template <typename W>
__global__ void __launch_bounds__(kSumThreads)
grad_weight_sum_kernel(const float* __restrict__ partial, int slabs, int dim, W* __restrict__ grad_weight,
                       W* __restrict__ grad_bias) {
  constexpr int kWarps = kSumThreads / 32;
  __shared__ float acc[kWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  W* to = blockIdx.y ? grad_bias : grad_weight;
  if (!to) return;
  const float* from = partial + (int64_t)blockIdx.y * slabs * dim;
  float sum = 0.f;
  if (c < dim) {
#pragma unroll 8
    for (int s = warp; s < slabs; s += kWarps) sum += from[(int64_t)s * dim + c];
  }
  acc[warp][lane] = sum;
  __syncthreads();
  sum = warp_sum(acc[lane][warp]);  // warp w adds up column w
  if (lane == 0 && blockIdx.x * 32 + warp < dim) to[blockIdx.x * 32 + warp] = narrow<W>(sum);
}

// ---------------------------------------------------------------------------
// Rows of more than 4096 elements: a CTA of THREADS per row, several passes over it
// (the later ones from L1 or L2), the weight's gradient by a kernel of its own.
//
// HBM-bound in many rows, bound by the passes' latency in few.  us, layer norm forward / backward, one warp per
// row and one element per load before: 4096 x 8192 bf16 38 / 86 (92 / 240; 3.5 and 2.3 TB/s), 16384 x 5120 fp32
// 198 / 345 (311 / 817), 32 x 8192 bf16 4 / 13 (51 / 71), 1 x 2^20 bf16 106 / 356 (6332 / 7966).
// ---------------------------------------------------------------------------
template <int E, typename F>
__device__ __forceinline__ void each_pack(int dim, int threads, F f) {
#pragma unroll 4
  for (int c = threadIdx.x * E; c < dim; c += threads * E) f(c);
}

template <typename T, int KIND, int E, int THREADS>
__global__ void __launch_bounds__(THREADS)
forward_wide_kernel(const T* __restrict__ tokens, const __grid_constant__ Rows t, Affine weight, Affine bias,
                    T* __restrict__ out, float* __restrict__ mean, float* __restrict__ rstd, float eps) {
  using X = Elem<E>;
  constexpr int N = kElems<E>;
  __shared__ float words[THREADS / 8];
  Team<THREADS> team(words);
  const float per = 1.0f / t.dim, least = least_square(eps);
  const Turn<THREADS> turn(t);
  Walker here;
  if (turn.begin < turn.end) here.find(t, turn.begin);
  for (int32_t row = turn.begin; row < turn.end; ++row) {
    here.seek(t, row);
    const T* const x = tokens + here.from(t, row);
    T* const y = out + (int64_t)row * t.dim;
    X sum = splat<X>(0.f);
    each_pack<E>(t.dim, THREADS, [&](int c) {
      X f[N];
      expand(load_pack<T, E>(x + c), f);
#pragma unroll
      for (int i = 0; i < N; ++i) sum = KIND == kLayer ? add(f[i], sum) : fma(f[i], f[i], sum);
    });
    const float first = team.sum(total(sum));
    if constexpr (KIND == kLayer) {
      const float mu = first * per;
      const X minus_mu = splat<X>(-mu);
      sum = splat<X>(0.f);
      each_pack<E>(t.dim, THREADS, [&](int c) {
        X f[N];
        expand(load_pack<T, E>(x + c), f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const X d = add(f[i], minus_mu);
          sum = fma(d, d, sum);
        }
      });
      const float r = rsqrtf(team.sum(total(sum)) * per + eps);
      const X rr = splat<X>(r);
      each_pack<E>(t.dim, THREADS, [&](int c) {
        X f[N], w[N], b[N];
        expand(load_pack<T, E>(x + c), f);
        if (weight.p) weight.pack<T, E>(c, w);
        if (bias.p) bias.pack<T, E>(c, b);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          f[i] = mul(add(f[i], minus_mu), rr);
          if (weight.p) f[i] = mul(f[i], w[i]);
          if (bias.p) f[i] = add(f[i], b[i]);
        }
        store_pack<T, E>(y + c, compress<T, E>(f));
      });
      if (mean && threadIdx.x == 0) {
        mean[row] = mu;
        rstd[row] = r;
      }
    } else {
      float ss = first, inv = rsqrtf(ss);
      float2 by = make_float2(1.f, 1.f);
      if (!plain_square(ss, least)) {
        float top = 0.f;
        each_pack<E>(t.dim, THREADS, [&](int c) {
          X f[N];
          expand(load_pack<T, E>(x + c), f);
#pragma unroll
          for (int i = 0; i < N; ++i) top = fmaxf(top, most(f[i]));
        });
        top = team.max(top);
        if (top > 0.f && top < INFINITY) {
          by = reciprocal_parts(top);
          sum = splat<X>(0.f);
          each_pack<E>(t.dim, THREADS, [&](int c) {
            X f[N];
            expand(load_pack<T, E>(x + c), f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const X d = mul(mul(f[i], splat<X>(by.x)), splat<X>(by.y));
              sum = fma(d, d, sum);
            }
          });
          ss = team.sum(total(sum));
        }
        const UnitScale u = unit_scale(ss, top, eps);
        inv = u.inv;
        if (!u.scaled) by = make_float2(1.f, 1.f);
      }
      each_pack<E>(t.dim, THREADS, [&](int c) {
        X f[N];
        expand(load_pack<T, E>(x + c), f);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = mul(mul(mul(f[i], splat<X>(by.x)), splat<X>(by.y)), splat<X>(inv));
        store_pack<T, E>(y + c, compress<T, E>(f));
      });
    }
  }
}

// grad_tokens.
template <typename T, int KIND, int E, int THREADS>
__global__ void __launch_bounds__(THREADS)
backward_wide_kernel(const T* __restrict__ grad, const T* __restrict__ tokens, const __grid_constant__ Rows t,
                     Affine weight, const float* __restrict__ mean, const float* __restrict__ rstd,
                     T* __restrict__ grad_tokens, float eps) {
  using X = Elem<E>;
  constexpr int N = kElems<E>;
  __shared__ float words[THREADS / 8];
  Team<THREADS> team(words);
  const float per = 1.0f / t.dim, least = least_square(eps);
  const Turn<THREADS> turn(t);
  Walker here;
  if (t.offsets) zero_padding<T, E>(t, grad_tokens, blockIdx.x, gridDim.x, threadIdx.x, THREADS);
  if (turn.begin < turn.end) here.find(t, turn.begin);
  for (int32_t row = turn.begin; row < turn.end; ++row) {
    here.seek(t, row);
    const T* const x = tokens + here.from(t, row);
    const T* const g = grad + (int64_t)row * t.dim;
    T* const dx = grad_tokens + here.slot(t, row) * t.dim;
    const auto packs_of = [&](int c, X (&f)[N], X (&d)[N]) {
      expand(load_pack<T, E>(x + c), f);
      expand(load_pack<T, E>(g + c), d);
    };
    if constexpr (KIND == kLayer) {
      const float r = rstd[row];
      const X minus_mu = splat<X>(-mean[row]), rr = splat<X>(r);
      X su = splat<X>(0.f), suh = su;
      each_pack<E>(t.dim, THREADS, [&](int c) {
        X f[N], u[N], w[N];
        packs_of(c, f, u);
        if (weight.p) weight.pack<T, E>(c, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (weight.p) u[i] = mul(u[i], w[i]);
          su = add(u[i], su);
          suh = fma(u[i], mul(add(f[i], minus_mu), rr), suh);
        }
      });
      const float2 both = team.sums(total(su), total(suh));
      const X minus_u = splat<X>(-r * (both.x * per)), minus_h = splat<X>(-r * (both.y * per));
      each_pack<E>(t.dim, THREADS, [&](int c) {
        X f[N], u[N], w[N];
        packs_of(c, f, u);
        if (weight.p) weight.pack<T, E>(c, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (weight.p) u[i] = mul(u[i], w[i]);
          f[i] = fma(u[i], rr, fma(mul(add(f[i], minus_mu), rr), minus_h, minus_u));
        }
        store_pack<T, E>(dx + c, compress<T, E>(f));
      });
    } else {
      X squares = splat<X>(0.f), products = squares;
      each_pack<E>(t.dim, THREADS, [&](int c) {
        X f[N], d[N];
        packs_of(c, f, d);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          squares = fma(f[i], f[i], squares);
          products = fma(f[i], d[i], products);
        }
      });
      float2 both = team.sums(total(squares), total(products));
      float inv = rsqrtf(both.x), along = both.y * inv;  // along: y . g
      float2 by = make_float2(1.f, 1.f);
      if (!plain_square(both.x, least)) {
        float top = 0.f;
        each_pack<E>(t.dim, THREADS, [&](int c) {
          X f[N];
          expand(load_pack<T, E>(x + c), f);
#pragma unroll
          for (int i = 0; i < N; ++i) top = fmaxf(top, most(f[i]));
        });
        top = team.max(top);
        if (top > 0.f && top < INFINITY) {
          by = reciprocal_parts(top);
          squares = products = splat<X>(0.f);
          each_pack<E>(t.dim, THREADS, [&](int c) {
            X f[N], d[N];
            packs_of(c, f, d);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              f[i] = mul(mul(f[i], splat<X>(by.x)), splat<X>(by.y));
              squares = fma(f[i], f[i], squares);
              products = fma(f[i], d[i], products);
            }
          });
          both = team.sums(total(squares), total(products));
        }
        const UnitScale u = unit_scale(both.x, top, eps);
        inv = u.inv;
        along = u.clamped ? 0.0f : both.y * inv;
        if (!u.scaled) by = make_float2(1.f, 1.f);
      }
      const X minus = splat<X>(-along), ii = splat<X>(inv), bx = splat<X>(by.x), bw = splat<X>(by.y);
      each_pack<E>(t.dim, THREADS, [&](int c) {
        X f[N], d[N];
        packs_of(c, f, d);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const X h = mul(mul(mul(f[i], bx), bw), ii);
          f[i] = mul(mul(mul(fma(h, minus, d[i]), ii), bx), bw);
        }
        store_pack<T, E>(dx + c, compress<T, E>(f));
      });
    }
  }
}

// Partial sums of grad_weight and grad_bias: a thread takes one pack of columns of one slab
// of consecutive rows, four rows at a time.  partial [2][slabs][dim].
template <typename T, int E>
__global__ void __launch_bounds__(kThreads)
grad_weight_wide_kernel(const T* __restrict__ grad, const T* __restrict__ tokens, const __grid_constant__ Rows t,
                        const float* __restrict__ mean, const float* __restrict__ rstd,
                        float* __restrict__ partial, int slabs) {
  using X = Elem<E>;
  constexpr int N = kElems<E>, kAtOnce = 4;
  const int c = (blockIdx.x * kThreads + threadIdx.x) * E;
  const int64_t used = t.used(), share = (used + slabs - 1) / slabs;
  const int32_t begin = (int32_t)min(blockIdx.y * share, used), end = (int32_t)min(begin + share, used);
  Walker here;
  if (begin < end) here.find(t, begin);
  if (c >= t.dim) return;
  X dw[N], db[N];
#pragma unroll
  for (int i = 0; i < N; ++i) dw[i] = db[i] = splat<X>(0.f);
  for (int32_t row = begin; row < end; row += kAtOnce) {
    Pack<T, E> x[kAtOnce], g[kAtOnce];
    float mu[kAtOnce], r[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (row + k >= end) break;
      here.seek(t, row + k);
      x[k] = load_pack<T, E>(tokens + here.from(t, row + k) + c);
      g[k] = load_pack<T, E>(grad + (int64_t)(row + k) * t.dim + c);
      mu[k] = mean[row + k];
      r[k] = rstd[row + k];
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (row + k >= end) break;
      X f[N], d[N];
      expand(x[k], f);
      expand(g[k], d);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        dw[i] = fma(d[i], mul(add(f[i], splat<X>(-mu[k])), splat<X>(r[k])), dw[i]);
        db[i] = add(d[i], db[i]);
      }
    }
  }
  const Pack<float, E> pw = unpacked<E>(dw), pb = unpacked<E>(db);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    partial[(int64_t)blockIdx.y * t.dim + c + e] = pw.v[e];
    partial[((int64_t)slabs + blockIdx.y) * t.dim + c + e] = pb.v[e];
  }
}

}  // namespace norm
}  // namespace maxsim
