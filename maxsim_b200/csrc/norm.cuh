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

// Which rows there are, where a row is read and which packed row it is.
struct Rows {
  int64_t segment_stride, row_stride;  // of the token rows, in elements
  const int32_t* offsets;              // [n_segments + 1], or null: every row counts
  int64_t packed_rows;                 // rows at or beyond are never touched
  uint32_t n_slots, L_max;             // n_slots = n_segments * L_max
  int dim;
};

struct Place {
  int64_t from;  // first element of the token row
  int64_t to;    // packed row, -1 for padding
};

__device__ __forceinline__ Place place_of(const Rows& t, uint32_t slot) {
  const uint32_t n = slot / t.L_max, j = slot - n * t.L_max;
  Place p;
  p.from = (int64_t)n * t.segment_stride + (int64_t)j * t.row_stride;
  p.to = slot;
  if (t.offsets) {
    const int64_t o0 = __ldg(t.offsets + n), o1 = __ldg(t.offsets + n + 1);
    p.to = o0 + j;
    if (o0 < 0 || p.to >= o1 || p.to >= t.packed_rows) p.to = -1;
  }
  return p;
}

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

// The factors of a unit row: y_i = (x_i * pre) * inv.  A sum of squares near the
// ends of the 32-bit range is taken again over x / max|x| (pre = 1 / max|x|).
struct UnitScale {
  float pre, inv;
  bool clamped;  // |x| <= eps: y = x / eps
};
__device__ __forceinline__ bool squares_out_of_range(float ss) { return ss > 1e37f || ss < 1e-30f; }
__device__ __forceinline__ UnitScale unit_scale(float ss, float top, bool scaled, float eps) {
  // |x| = top * sqrt(ss) when scaled by top, else sqrt(ss); a NaN stays one
  const float norm = scaled ? top * sqrtf(ss) : sqrtf(ss);
  UnitScale u;
  if (norm == INFINITY && !scaled) {  // an infinity in the row: finite / inf = 0, inf / inf = NaN
    u.pre = 1.0f;
    u.inv = 0.0f;
    u.clamped = false;
    return u;
  }
  u.clamped = norm <= eps;
  u.pre = scaled && !u.clamped ? 1.0f / top : 1.0f;
  u.inv = u.clamped ? 1.0f / eps : 1.0f / sqrtf(ss);
  return u;
}

// One warp per row, three passes over it.
template <typename T, typename W, int KIND>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const T* __restrict__ tokens, Rows t, const W* __restrict__ weight,
               const W* __restrict__ bias, T* __restrict__ out, float* __restrict__ mean,
               float* __restrict__ rstd, float eps) {
  const int lane = threadIdx.x & 31;
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint32_t slot = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); slot < t.n_slots; slot += warps) {
    const Place p = place_of(t, slot);
    if (p.to < 0) continue;
    const T* x = tokens + p.from;
    T* y = out + p.to * t.dim;
    if (KIND == kLayer) {
      float s = 0.f;
      for (int c = lane; c < t.dim; c += 32) s += widen(x[c]);
      const float mu = warp_sum(s) / t.dim;
      float ss = 0.f;
      for (int c = lane; c < t.dim; c += 32) {
        const float d = widen(x[c]) - mu;
        ss += d * d;
      }
      const float r = 1.0f / sqrtf(warp_sum(ss) / t.dim + eps);
      for (int c = lane; c < t.dim; c += 32) {
        float h = (widen(x[c]) - mu) * r;
        if (weight) h *= widen(weight[c]);
        if (bias) h += widen(bias[c]);
        y[c] = narrow<T>(h);
      }
      if (mean && lane == 0) {
        mean[p.to] = mu;
        rstd[p.to] = r;
      }
    } else {
      float ss = 0.f, top = 0.f;
      for (int c = lane; c < t.dim; c += 32) {
        const float v = widen(x[c]);
        ss += v * v;
        top = fmaxf(top, fabsf(v));
      }
      ss = warp_sum(ss);
      top = warp_max(top);
      const bool scaled = squares_out_of_range(ss) && top > 0.f && top < INFINITY;
      if (scaled) {
        ss = 0.f;
        for (int c = lane; c < t.dim; c += 32) {
          const float v = widen(x[c]) / top;
          ss += v * v;
        }
        ss = warp_sum(ss);
      }
      const UnitScale u = unit_scale(ss, top, scaled, eps);
      for (int c = lane; c < t.dim; c += 32) y[c] = narrow<T>(widen(x[c]) * u.pre * u.inv);
    }
  }
}

// grad_tokens.  One warp per row; the gradient of a padding row is zero.
template <typename T, typename W, int KIND>
__global__ void __launch_bounds__(kThreads)
backward_kernel(const T* __restrict__ grad, const T* __restrict__ tokens, Rows t,
                const W* __restrict__ weight, const float* __restrict__ mean,
                const float* __restrict__ rstd, T* __restrict__ grad_tokens, float eps) {
  const int lane = threadIdx.x & 31;
  const uint32_t warps = gridDim.x * (kThreads / 32);
  for (uint32_t slot = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); slot < t.n_slots; slot += warps) {
    const Place p = place_of(t, slot);
    T* dx = grad_tokens + (int64_t)slot * t.dim;
    if (p.to < 0) {
      for (int c = lane; c < t.dim; c += 32) dx[c] = narrow<T>(0.f);
      continue;
    }
    const T* x = tokens + p.from;
    const T* g = grad + p.to * t.dim;
    if (KIND == kLayer) {
      const float mu = mean[p.to], r = rstd[p.to];
      float su = 0.f, suh = 0.f;
      for (int c = lane; c < t.dim; c += 32) {
        const float u = widen(g[c]) * (weight ? widen(weight[c]) : 1.0f);
        su += u;
        suh += u * ((widen(x[c]) - mu) * r);
      }
      su = warp_sum(su) / t.dim;
      suh = warp_sum(suh) / t.dim;
      for (int c = lane; c < t.dim; c += 32) {
        const float u = widen(g[c]) * (weight ? widen(weight[c]) : 1.0f);
        dx[c] = narrow<T>(r * (u - su - (widen(x[c]) - mu) * r * suh));
      }
    } else {
      float ss = 0.f, xg = 0.f, top = 0.f;
      for (int c = lane; c < t.dim; c += 32) {
        const float v = widen(x[c]);
        ss += v * v;
        xg += v * widen(g[c]);
        top = fmaxf(top, fabsf(v));
      }
      ss = warp_sum(ss);
      xg = warp_sum(xg);
      top = warp_max(top);
      const bool scaled = squares_out_of_range(ss) && top > 0.f && top < INFINITY;
      if (scaled) {
        ss = xg = 0.f;
        for (int c = lane; c < t.dim; c += 32) {
          const float v = widen(x[c]) / top;
          ss += v * v;
          xg += v * widen(g[c]);
        }
        ss = warp_sum(ss);
        xg = warp_sum(xg);
      }
      const UnitScale u = unit_scale(ss, top, scaled, eps);
      const float along = u.clamped ? 0.0f : xg * u.inv;  // y . g
      for (int c = lane; c < t.dim; c += 32) {
        const float h = widen(x[c]) * u.pre * u.inv;
        dx[c] = narrow<T>((widen(g[c]) - h * along) * u.inv * u.pre);
      }
    }
  }
}

// Partial sums of grad_weight and grad_bias: thread = one column of one slab
// of rows; slab s covers slots s, s + slabs, ...  partial [2][slabs][dim].
template <typename T>
__global__ void __launch_bounds__(kThreads)
grad_weight_kernel(const T* __restrict__ grad, const T* __restrict__ tokens, Rows t,
                   const float* __restrict__ mean, const float* __restrict__ rstd,
                   float* __restrict__ partial, int slabs) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= t.dim) return;
  float dw = 0.f, db = 0.f;
  for (uint32_t slot = blockIdx.y; slot < t.n_slots; slot += slabs) {
    const Place p = place_of(t, slot);
    if (p.to < 0) continue;
    const float g = widen(grad[p.to * t.dim + c]);
    dw += g * ((widen(tokens[p.from + c]) - mean[p.to]) * rstd[p.to]);
    db += g;
  }
  partial[(int64_t)blockIdx.y * t.dim + c] = dw;
  partial[((int64_t)slabs + blockIdx.y) * t.dim + c] = db;
}

template <typename W>
__global__ void __launch_bounds__(kThreads)
grad_weight_sum_kernel(const float* __restrict__ partial, int slabs, int dim, W* __restrict__ grad_weight,
                       W* __restrict__ grad_bias) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= dim) return;
  float dw = 0.f, db = 0.f;
  for (int s = 0; s < slabs; ++s) {
    dw += partial[(int64_t)s * dim + c];
    db += partial[((int64_t)slabs + s) * dim + c];
  }
  if (grad_weight) grad_weight[c] = narrow<W>(dw);
  if (grad_bias) grad_bias[c] = narrow<W>(db);
}

}  // namespace norm
}  // namespace maxsim
