// extern "C" entry points of the row normalisation operators, and their dispatch.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <limits>

#include "host.h"
#include "norm.cuh"

namespace maxsim {
namespace {

constexpr int64_t kMaxRows = (1ll << 31) - 4096;  // 32-bit row counters run a few turns ahead

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of the partial sums of the weight's gradient: one for each CTA of a layer norm's
// backward kernel, at most 512 threads or four CTAs on an SM.
int grad_slabs(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(rows, 4 * sm_count())); }

// How the packed rows are split over a grid: every unit (a warp, or the CTA of a
// wide team) gets the same number of consecutive rows.
struct Split {
  unsigned grid;
  int32_t chunk;
  norm::Rows of(norm::Rows t) const {
    t.chunk = chunk;
    return t;
  }
};
template <int THREADS, int TEAM>
Split share_rows(int64_t rows, int ctas_per_sm) {
  constexpr int units = TEAM > 32 ? 1 : THREADS / 32, together = TEAM >= 32 ? 1 : 32 / TEAM;
  const int64_t most = (int64_t)sm_count() * ctas_per_sm * units;
  const int64_t chunk = ceil_div(ceil_div(rows, most), together) * together;
  return {(unsigned)ceil_div(ceil_div(rows, chunk), units), (int32_t)chunk};
}

struct Forward {
  static constexpr bool kSums = false;
  const void* tokens;
  norm::Rows t;
  norm::Affine weight, bias;
  void* out;
  float* mean;
  float* rstd;
  float eps;
  cudaStream_t st;
  const char* name() const { return "norm forward_rows_kernel"; }
  // Whether every row and vector starts on a multiple of `bytes`, strides aside.
  bool aligned(int bytes) const {
    const uintptr_t all = (uintptr_t)tokens | (uintptr_t)out | (uintptr_t)weight.p | (uintptr_t)bias.p;
    return all % bytes == 0;
  }

  template <typename T, int KIND, int E, int TEAM, int V>
  int rows() const {
    constexpr int threads = norm::kCtaThreads<TEAM>, per_sm = norm::kForwardThreads<E, TEAM, V>;
    constexpr int ring = norm::kRingBytes<T, E, TEAM, V, 1, per_sm>;
    auto kern = norm::forward_rows_kernel<T, KIND, E, TEAM, V>;
    static std::atomic<unsigned char> configured[kMaxDevices];
    constexpr int most = ring + (KIND == norm::kLayer ? 2 * norm::Wide<E>::bytes(TEAM * V * E) : 0);
    static_assert(most <= 227 * 1024, "shared memory of a CTA");
    if (int rc = ensure_smem(kern, most, configured)) return rc;
    const Split split = share_rows<threads, TEAM>(t.rows, per_sm / threads);
    const int smem = ring + (KIND == norm::kLayer ? 2 * norm::Wide<E>::bytes(t.dim) : 0);
    kern<<<split.grid, threads, smem, st>>>((const T*)tokens, split.of(t), weight, bias, (T*)out, mean, rstd, eps);
    return launch_check(name());
  }
  template <typename T, int KIND>
  int wide() const {
    const Split split = share_rows<norm::kThreads, 32>(t.rows, 8);
    norm::forward_wide_kernel<T, KIND><<<split.grid, norm::kThreads, 0, st>>>(
        (const T*)tokens, split.of(t), weight, bias, (T*)out, mean, rstd, eps);
    return launch_check("norm forward_wide_kernel");
  }
};

struct Backward {
  static constexpr bool kSums = true;
  const void* grad;
  const void* tokens;
  norm::Rows t;
  norm::Affine weight;
  const float* mean;
  const float* rstd;
  void* grad_tokens;
  float* partial;  // null: no sums are wanted
  float eps;
  cudaStream_t st;
  mutable int slabs = 0;  // rows of `partial` that were written
  bool aligned(int bytes) const {
    const uintptr_t all = (uintptr_t)grad | (uintptr_t)tokens | (uintptr_t)grad_tokens | (uintptr_t)weight.p;
    return all % bytes == 0;
  }

  template <typename T, int KIND, int E, int TEAM, int V>
  int rows() const {
    constexpr int threads = norm::kCtaThreads<TEAM>, per_sm = norm::kBackwardThreads<KIND, E, TEAM, V>;
    constexpr int fixed = norm::kBackwardBytes<T, KIND, E, TEAM, V>;
    auto kern = norm::backward_rows_kernel<T, KIND, E, TEAM, V>;
    static std::atomic<unsigned char> configured[kMaxDevices];
    constexpr int most = fixed + (KIND == norm::kLayer ? norm::Wide<E>::bytes(TEAM * V * E) : 0);
    static_assert(most <= 227 * 1024, "shared memory of a CTA");
    if (int rc = ensure_smem(kern, most, configured)) return rc;
    Split split = share_rows<threads, TEAM>(std::max(t.rows, 1), per_sm / threads);
    if (t.offsets) {  // few rows in much padding: as many CTAs as its zeros keep busy
      const int64_t most_ctas = (int64_t)sm_count() * (per_sm / threads);
      split.grid = (unsigned)std::max<int64_t>(split.grid, std::min(most_ctas, ceil_div((int64_t)t.n_segments * t.L_max, 64)));
    }
    slabs = (int)split.grid;
    const int smem = fixed + (KIND == norm::kLayer ? norm::Wide<E>::bytes(t.dim) : 0);
    kern<<<split.grid, threads, smem, st>>>((const T*)grad, (const T*)tokens, split.of(t), weight, mean, rstd,
                                            (T*)grad_tokens, partial, eps);
    return launch_check("norm backward_rows_kernel");
  }
  template <typename T, int KIND>
  int wide() const {
    if (grad_tokens) {
      const Split split = share_rows<norm::kThreads, 32>(std::max(t.rows, 1), 8);
      norm::backward_wide_kernel<T, KIND><<<split.grid, norm::kThreads, 0, st>>>(
          (const T*)grad, (const T*)tokens, split.of(t), weight, mean, rstd, (T*)grad_tokens, eps);
      if (int rc = launch_check("norm backward_wide_kernel")) return rc;
    }
    if (!partial) return MAXSIM_OK;
    slabs = std::min(grad_slabs(t.rows), 64);
    norm::grad_weight_wide_kernel<T><<<dim3((unsigned)ceil_div(t.dim, norm::kThreads), (unsigned)slabs),
                                       norm::kThreads, 0, st>>>(
        (const T*)grad, (const T*)tokens, t, mean, rstd, partial, slabs);
    return launch_check("norm grad_weight_wide_kernel");
  }
};

// The team a row gets.  Few threads with many packs cost fewer instructions a row (the
// shuffles and the bookkeeping are shared by 32 / TEAM rows), which is what the narrow rows and the
// forward pass are short of; the backward pass of a layer norm keeps two column sums
// for every element a thread holds and takes wider teams.
template <typename T, int KIND, int E, typename Call>
int by_width(const Call& call) {
  constexpr bool sums = Call::kSums && KIND == norm::kLayer;
  const int packs = (call.t.dim + E - 1) / E;
  if constexpr (E == 8) {
    if constexpr (KIND == norm::kUnit) {
      if (packs <= 2) return call.template rows<T, KIND, E, 2, 1>();
      if (packs <= 4) return call.template rows<T, KIND, E, 4, 1>();
    }
    if (packs <= 8) return call.template rows<T, KIND, E, 8, 1>();
    if (packs <= 16) return call.template rows<T, KIND, E, 8, 2>();
    if (packs <= 32) return call.template rows<T, KIND, E, 16, 2>();
    if constexpr (sums) {
      if (packs <= 64) return call.template rows<T, KIND, E, 32, 2>();
      if (packs <= 96) return call.template rows<T, KIND, E, 32, 3>();
    } else {
      if (packs <= 48) return call.template rows<T, KIND, E, 16, 3>();
      if (packs <= 64) return call.template rows<T, KIND, E, 16, 4>();
      if (packs <= 96) return call.template rows<T, KIND, E, 32, 3>();
    }
    if (packs <= 128) return call.template rows<T, KIND, E, 32, 4>();
    if (packs <= 256) return call.template rows<T, KIND, E, norm::kWide, 2>();
    if (packs <= 512) return call.template rows<T, KIND, E, norm::kWide, 4>();
  } else if constexpr (E == 4) {
    if (packs <= 8) return call.template rows<T, KIND, E, 8, 1>();
    if (packs <= 16) return call.template rows<T, KIND, E, 8, 2>();
    if (packs <= 32) return call.template rows<T, KIND, E, 8, 4>();
    if (packs <= 64) return call.template rows<T, KIND, E, 16, 4>();
    if (packs <= 128) return call.template rows<T, KIND, E, 32, 4>();
    if (packs <= 192) return call.template rows<T, KIND, E, 32, 6>();
    if (packs <= 256) return call.template rows<T, KIND, E, 32, 8>();
    if (packs <= 512) return call.template rows<T, KIND, E, norm::kWide, 4>();
    if (packs <= 1024) return call.template rows<T, KIND, E, norm::kWide, 8>();
  } else if constexpr (E == 2) {
    if (packs <= 16) return call.template rows<T, KIND, E, 8, 2>();
    if (packs <= 32) return call.template rows<T, KIND, E, 16, 2>();
    if (packs <= 64) return call.template rows<T, KIND, E, 16, 4>();
    if (packs <= 128) return call.template rows<T, KIND, E, 32, 4>();
    if (packs <= 192) return call.template rows<T, KIND, E, 32, 6>();
    if (packs <= 512) return call.template rows<T, KIND, E, 32, 16>();
    if (packs <= 768) return call.template rows<T, KIND, E, norm::kWide, 6>();
    if (packs <= 2048) return call.template rows<T, KIND, E, norm::kWide, 16>();
  } else {
    if (packs <= 32) return call.template rows<T, KIND, E, 32, 1>();
    if (packs <= 64) return call.template rows<T, KIND, E, 32, 2>();
    if (packs <= 96) return call.template rows<T, KIND, E, 32, 3>();
    if (packs <= 128) return call.template rows<T, KIND, E, 32, 4>();
    if (packs <= 256) return call.template rows<T, KIND, E, 32, 8>();
    if (packs <= 384) return call.template rows<T, KIND, E, 32, 12>();
    if constexpr (sums && sizeof(T) == 4) {
      if (packs <= 1024) return call.template rows<T, KIND, E, norm::kWide, 8>();
    }
    if (packs <= 1024) return call.template rows<T, KIND, E, 32, 32>();
    if (packs <= 4096) return call.template rows<T, KIND, E, norm::kWide, 32>();
  }
  return call.template wide<T, KIND>();
}

// The widest pack on whose multiples every row starts and ends.
template <typename T, int KIND, typename Call>
int by_alignment(const Call& call) {
  const norm::Rows& t = call.t;
  const int64_t all = t.dim | t.segment_stride | t.row_stride;
  if (call.aligned(16) && all % (16 / sizeof(T)) == 0) return by_width<T, KIND, 16 / sizeof(T)>(call);
  if constexpr (sizeof(T) == 2) {
    if (call.aligned(4) && all % 2 == 0) return by_width<T, KIND, 2>(call);
  }
  return by_width<T, KIND, 1>(call);
}

template <typename Call>
int launch(int kind, int dtype, const Call& call) {
  const bool layer = kind == norm::kLayer;
  switch (dtype) {
    case MAXSIM_F32:
      return layer ? by_alignment<float, norm::kLayer>(call) : by_alignment<float, norm::kUnit>(call);
    case MAXSIM_F16:
      return layer ? by_alignment<__half, norm::kLayer>(call) : by_alignment<__half, norm::kUnit>(call);
    default:
      return layer ? by_alignment<__nv_bfloat16, norm::kLayer>(call) : by_alignment<__nv_bfloat16, norm::kUnit>(call);
  }
}

template <typename W>
int launch_sum(const Backward& call, void* grad_weight, void* grad_bias) {
  norm::grad_weight_sum_kernel<W><<<dim3((unsigned)ceil_div(call.t.dim, 32), 2), norm::kSumThreads, 0, call.st>>>(
      call.partial, call.slabs, call.t.dim, (W*)grad_weight, (W*)grad_bias);
  return launch_check("norm grad_weight_sum_kernel");
}

int check_types(int dtype, int weight_dtype) {
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype)) return fail(MAXSIM_EINVAL, "unknown dtype code");
  if (weight_dtype != dtype && weight_dtype != MAXSIM_F32)
    return fail(MAXSIM_EUNSUPPORTED, "weights must be float or of the tokens' type");
  return MAXSIM_OK;
}

int check_rows(int kind, int64_t n_segments, int64_t L_max, int64_t dim, int64_t packed_rows,
               int64_t segment_stride, int64_t row_stride, const int32_t* offsets, double eps, norm::Rows* t) {
  if (kind != norm::kLayer && kind != norm::kUnit) return fail(MAXSIM_EINVAL, "unknown norm code %d", kind);
  if (n_segments < 0 || L_max < 0 || dim <= 0 || packed_rows < 0)
    return fail(MAXSIM_EINVAL, "sizes must not be negative, dim must be positive");
  if (dim > (1ll << 24)) return fail(MAXSIM_EUNSUPPORTED, "dim=%lld too large", (long long)dim);
  if (n_segments > kMaxRows || L_max > kMaxRows || (L_max && n_segments > kMaxRows / L_max)) return fail(MAXSIM_EUNSUPPORTED, "at most 2^31 - 4096 rows");
  if (segment_stride < 0 || row_stride < 0) return fail(MAXSIM_EINVAL, "strides must not be negative");
  if (!(eps > 0.0) || !std::isfinite((float)eps) || (float)eps < 1e-30f)
    return fail(MAXSIM_EINVAL, "eps must be at least 1e-30; got %g", eps);
  t->segment_stride = segment_stride;
  t->row_stride = row_stride;
  t->offsets = offsets;
  t->n_segments = (int32_t)n_segments;
  t->L_max = (int32_t)L_max;
  // more packed rows than token rows cannot be filled
  t->rows = (int32_t)std::min(packed_rows, n_segments * L_max);
  t->chunk = 0;
  t->dim = (int32_t)dim;
  return MAXSIM_OK;
}

}  // namespace
}  // namespace maxsim

using namespace maxsim;

extern "C" {

int maxsim_b200_norm_rows(int kind, const void* tokens, int64_t segment_stride, int64_t row_stride,
                          const int32_t* offsets, const void* weight, const void* bias, void* out, float* mean,
                          float* rstd, int64_t n_segments, int64_t L_max, int64_t dim, int64_t packed_rows,
                          double eps, int dtype, int weight_dtype, void* stream) {
  norm::Rows t;
  if (int rc = check_rows(kind, n_segments, L_max, dim, packed_rows, segment_stride, row_stride, offsets, eps, &t))
    return rc;
  if (int rc = check_types(dtype, weight_dtype)) return rc;
  if (t.rows == 0) return MAXSIM_OK;
  if (!tokens || !out) return fail(MAXSIM_EINVAL, "null pointer argument");
  if ((mean == nullptr) != (rstd == nullptr)) return fail(MAXSIM_EINVAL, "mean and rstd come together");
  if (kind == norm::kUnit && (weight || bias)) return fail(MAXSIM_EINVAL, "unit rows have no weights");
  const bool f32 = weight_dtype == MAXSIM_F32;
  return launch(kind, dtype, Forward{tokens, t, {weight, f32}, {bias, f32}, out, mean, rstd, (float)eps,
                                     static_cast<cudaStream_t>(stream)});
}

int64_t maxsim_b200_norm_rows_workspace(int64_t n_segments, int64_t L_max, int64_t dim) {
  if (n_segments <= 0 || L_max <= 0 || dim <= 0 || n_segments > kMaxRows / L_max) return 0;
  return (int64_t)grad_slabs(n_segments * L_max) * dim * 2 * (int64_t)sizeof(float);
}

int maxsim_b200_norm_rows_backward(int kind, const void* grad, const void* tokens, int64_t segment_stride,
                                   int64_t row_stride, const int32_t* offsets, const void* weight,
                                   const float* mean, const float* rstd, void* grad_tokens, void* grad_weight,
                                   void* grad_bias, void* workspace, int64_t workspace_bytes,
                                   int64_t n_segments, int64_t L_max, int64_t dim, int64_t packed_rows,
                                   double eps, int dtype, int weight_dtype, void* stream) {
  norm::Rows t;
  if (int rc = check_rows(kind, n_segments, L_max, dim, packed_rows, segment_stride, row_stride, offsets, eps, &t))
    return rc;
  if (kind == norm::kUnit && (weight || grad_weight || grad_bias))
    return fail(MAXSIM_EINVAL, "unit rows have no weights");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool sums = grad_weight || grad_bias;
  if (int rc = check_types(dtype, weight_dtype)) return rc;
  if (n_segments * L_max == 0) {  // no rows: the sums are zero
    const size_t bytes = (size_t)dim * (weight_dtype == MAXSIM_F32 ? 4 : 2);
    if (grad_weight) MAXSIM_CUDA(cudaMemsetAsync(grad_weight, 0, bytes, st));
    if (grad_bias) MAXSIM_CUDA(cudaMemsetAsync(grad_bias, 0, bytes, st));
    return MAXSIM_OK;
  }
  if (!grad_tokens && !sums) return MAXSIM_OK;
  if (!tokens || (!grad && packed_rows > 0)) return fail(MAXSIM_EINVAL, "null pointer argument");
  if (kind == norm::kLayer && packed_rows > 0 && (!mean || !rstd)) return fail(MAXSIM_EINVAL, "null pointer argument");
  if (sums && (!workspace || workspace_bytes < maxsim_b200_norm_rows_workspace(n_segments, L_max, dim)))
    return fail(MAXSIM_EWORKSPACE, "workspace missing or smaller than maxsim_b200_norm_rows_workspace says");
  const Backward call{grad, tokens, t, {weight, weight_dtype == MAXSIM_F32}, mean, rstd, grad_tokens,
                      sums ? static_cast<float*>(workspace) : nullptr, (float)eps, st};
  if (int rc = launch(kind, dtype, call)) return rc;
  if (!sums) return MAXSIM_OK;
  switch (weight_dtype) {
    case MAXSIM_F32: return launch_sum<float>(call, grad_weight, grad_bias);
    case MAXSIM_F16: return launch_sum<__half>(call, grad_weight, grad_bias);
    default: return launch_sum<__nv_bfloat16>(call, grad_weight, grad_bias);
  }
}

}  // extern "C"
