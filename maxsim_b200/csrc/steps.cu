// extern "C" entry points of the row normalisation and sampling operators, and
// their dispatch.  A translation unit of its own so that it builds beside
// abi.cu.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "host.h"
#include "norm.cuh"
#include "sample.cuh"

namespace maxsim {
namespace {

constexpr int64_t kMaxSlots = (1ll << 31) - 1;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int grad_slabs(int64_t slots, int64_t dim) {
  (void)dim;
  return (int)std::max<int64_t>(1, std::min<int64_t>(slots / 16, 4 * sm_count()));
}

template <typename T, typename W, int KIND>
int launch_forward(const void* tokens, const norm::Rows& t, const void* weight, const void* bias, void* out,
                   float* mean, float* rstd, float eps, cudaStream_t st) {
  const int64_t grid = std::min<int64_t>(ceil_div(t.n_slots, norm::kThreads / 32), (int64_t)sm_count() * 8);
  norm::forward_kernel<T, W, KIND><<<(unsigned)grid, norm::kThreads, 0, st>>>(
      (const T*)tokens, t, (const W*)weight, (const W*)bias, (T*)out, mean, rstd, eps);
  return launch_check("norm forward_kernel");
}

struct Grads {
  const void* grad;
  const float* mean;
  const float* rstd;
  void* tokens;
  void* weight;
  void* bias;
  float* partial;
};

template <typename T, typename W, int KIND>
int launch_backward(const void* tokens, const norm::Rows& t, const void* weight, const Grads& g, float eps,
                    cudaStream_t st) {
  if (g.tokens) {
    const int64_t grid = std::min<int64_t>(ceil_div(t.n_slots, norm::kThreads / 32), (int64_t)sm_count() * 8);
    norm::backward_kernel<T, W, KIND><<<(unsigned)grid, norm::kThreads, 0, st>>>(
        (const T*)g.grad, (const T*)tokens, t, (const W*)weight, g.mean, g.rstd, (T*)g.tokens, eps);
    if (int rc = launch_check("norm backward_kernel")) return rc;
  }
  if (KIND == norm::kLayer && (g.weight || g.bias)) {
    const int slabs = grad_slabs(t.n_slots, t.dim);
    const unsigned cols = (unsigned)ceil_div(t.dim, norm::kThreads);
    norm::grad_weight_kernel<T><<<dim3(cols, (unsigned)slabs), norm::kThreads, 0, st>>>(
        (const T*)g.grad, (const T*)tokens, t, g.mean, g.rstd, g.partial, slabs);
    if (int rc = launch_check("norm grad_weight_kernel")) return rc;
    norm::grad_weight_sum_kernel<W><<<cols, norm::kThreads, 0, st>>>(g.partial, slabs, t.dim, (W*)g.weight,
                                                                    (W*)g.bias);
    return launch_check("norm grad_weight_sum_kernel");
  }
  return MAXSIM_OK;
}

// Calls f(T{}, W{}): the token type and the weights' type, which is the same or float.
template <typename F>
int with_types(int dtype, int weight_dtype, F f) {
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype)) return fail(MAXSIM_EINVAL, "unknown dtype code");
  if (weight_dtype != dtype && weight_dtype != MAXSIM_F32)
    return fail(MAXSIM_EUNSUPPORTED, "weights must be float or of the tokens' type");
  if (dtype == MAXSIM_F32) return f(float{}, float{});
  if (dtype == MAXSIM_F16) return weight_dtype == MAXSIM_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
  return weight_dtype == MAXSIM_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

int check_rows(int kind, int64_t n_segments, int64_t L_max, int64_t dim, int64_t packed_rows,
               int64_t segment_stride, int64_t row_stride, const int32_t* offsets, double eps, norm::Rows* t) {
  if (kind != norm::kLayer && kind != norm::kUnit) return fail(MAXSIM_EINVAL, "unknown norm code %d", kind);
  if (n_segments < 0 || L_max < 0 || dim <= 0 || packed_rows < 0)
    return fail(MAXSIM_EINVAL, "sizes must not be negative, dim must be positive");
  if (dim > (1ll << 24)) return fail(MAXSIM_EUNSUPPORTED, "dim=%lld too large", (long long)dim);
  if (L_max && n_segments > kMaxSlots / L_max) return fail(MAXSIM_EUNSUPPORTED, "at most 2^31 - 1 rows");
  if (segment_stride < 0 || row_stride < 0) return fail(MAXSIM_EINVAL, "strides must not be negative");
  if (!(eps > 0.0) || !std::isfinite((float)eps) || (float)eps < 1e-30f)
    return fail(MAXSIM_EINVAL, "eps must be at least 1e-30; got %g", eps);
  t->segment_stride = segment_stride;
  t->row_stride = row_stride;
  t->offsets = offsets;
  t->packed_rows = packed_rows;
  t->n_slots = (uint32_t)(n_segments * L_max);
  t->L_max = (uint32_t)L_max;
  t->dim = (int)dim;
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
  if (t.n_slots == 0 || (offsets && packed_rows == 0)) return MAXSIM_OK;
  if (!tokens || !out) return fail(MAXSIM_EINVAL, "null pointer argument");
  if ((mean == nullptr) != (rstd == nullptr)) return fail(MAXSIM_EINVAL, "mean and rstd come together");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_types(dtype, weight_dtype, [&](auto a, auto b) {
    using T = decltype(a);
    using W = decltype(b);
    if (kind == norm::kLayer)
      return launch_forward<T, W, norm::kLayer>(tokens, t, weight, bias, out, mean, rstd, (float)eps, st);
    return launch_forward<T, W, norm::kUnit>(tokens, t, weight, bias, out, mean, rstd, (float)eps, st);
  });
}

int64_t maxsim_b200_norm_rows_workspace(int64_t n_segments, int64_t L_max, int64_t dim) {
  if (n_segments <= 0 || L_max <= 0 || dim <= 0 || n_segments > kMaxSlots / L_max) return 0;
  return (int64_t)grad_slabs(n_segments * L_max, dim) * dim * 2 * (int64_t)sizeof(float);
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
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype)) return fail(MAXSIM_EINVAL, "unknown dtype code");
  if (t.n_slots == 0) {  // no rows: the sums are zero
    const size_t bytes = (size_t)dim * (weight_dtype == MAXSIM_F32 ? 4 : 2);
    if (grad_weight) MAXSIM_CUDA(cudaMemsetAsync(grad_weight, 0, bytes, st));
    if (grad_bias) MAXSIM_CUDA(cudaMemsetAsync(grad_bias, 0, bytes, st));
    return MAXSIM_OK;
  }
  if (!tokens || (!grad && packed_rows > 0)) return fail(MAXSIM_EINVAL, "null pointer argument");
  if (kind == norm::kLayer && packed_rows > 0 && (!mean || !rstd)) return fail(MAXSIM_EINVAL, "null pointer argument");
  if (sums && (!workspace || workspace_bytes < maxsim_b200_norm_rows_workspace(n_segments, L_max, dim)))
    return fail(MAXSIM_EWORKSPACE, "workspace missing or smaller than maxsim_b200_norm_rows_workspace says");
  const Grads g{grad, mean, rstd, grad_tokens, grad_weight, grad_bias, static_cast<float*>(workspace)};
  return with_types(dtype, weight_dtype, [&](auto a, auto b) {
    using T = decltype(a);
    using W = decltype(b);
    if (kind == norm::kLayer) return launch_backward<T, W, norm::kLayer>(tokens, t, weight, g, (float)eps, st);
    return launch_backward<T, W, norm::kUnit>(tokens, t, weight, g, (float)eps, st);
  });
}

int maxsim_b200_sample_rows(const float* scores, int64_t score_stride, const float* uniforms,
                            int64_t uniform_stride, int64_t rows, int64_t cols, int64_t n, double temperature,
                            const float* temperature_rows, int64_t top_k, const int32_t* top_k_rows, double top_p,
                            const float* top_p_rows, double min_p, const float* min_p_rows, int64_t* indices,
                            float* probabilities, void* stream) {
  if (rows < 0 || cols < 0 || n < 0 || n > cols) return fail(MAXSIM_EINVAL, "need rows >= 0 and 0 <= n <= cols");
  if (rows >= (1ll << 31)) return fail(MAXSIM_EINVAL, "too many rows");
  if (cols > (1 << 20)) return fail(MAXSIM_EUNSUPPORTED, "at most 2^20 columns per row; got %lld", (long long)cols);
  if (n > 1024) return fail(MAXSIM_EUNSUPPORTED, "at most 1024 draws per row; got %lld", (long long)n);
  if (score_stride < 0 || uniform_stride < 0) return fail(MAXSIM_EINVAL, "strides must not be negative");
  if (!temperature_rows && !(temperature > 0.0)) return fail(MAXSIM_EINVAL, "temperature must be > 0");
  if (rows == 0 || n == 0) return MAXSIM_OK;
  if (!scores || !uniforms || !indices || !probabilities) return fail(MAXSIM_EINVAL, "null pointer argument");
  sample::Args A;
  A.scores = scores;
  A.uniforms = uniforms;
  A.score_stride = score_stride;
  A.uniform_stride = uniform_stride;
  A.rows = rows;
  A.cols = (int)cols;
  A.n = (int)n;
  A.temperature = {temperature, temperature_rows};
  A.top_p = {top_p, top_p_rows};
  A.min_p = {min_p, min_p_rows};
  A.top_k = {top_k, top_k_rows};
  A.shift = 62;
  for (int64_t c = 1; c < cols; c <<= 1) --A.shift;
  A.indices = indices;
  A.probabilities = probabilities;
  sample::sample_rows_kernel<<<(unsigned)rows, sample::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(A);
  return launch_check("sample_rows_kernel");
}

}  // extern "C"
