// extern "C" entry points of the gradients of the row normalisation operators.
#include "norm_host.cuh"

namespace maxsim {
namespace {

// Rows of the partial sums of the weight's gradient that a workspace holds: one for each CTA of a
// layer norm's backward kernel, which never has more CTAs than there are token rows.
int64_t grad_slabs(int64_t rows) { return std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t)norm::kSumCtas * sm_count())); }
int64_t workspace_bytes_for(int64_t slabs, int64_t dim) { return slabs * dim * 2 * (int64_t)sizeof(float); }

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
  int64_t partial_bytes;
  float eps;
  cudaStream_t st;
  mutable int slabs = 0;  // rows of `partial` that were written
  bool aligned(int bytes) const {
    const uintptr_t all = (uintptr_t)grad | (uintptr_t)tokens | (uintptr_t)grad_tokens | (uintptr_t)weight.p;
    return all % bytes == 0;
  }

  // Before a kernel that writes `n` rows of partial sums: that there is room for them.
  int take_slabs(int64_t n) const {
    slabs = (int)n;
    if (partial && workspace_bytes_for(n, t.dim) > partial_bytes)
      return fail(MAXSIM_EWORKSPACE, "%lld rows of partial sums do not fit the workspace", (long long)n);
    return MAXSIM_OK;
  }
  // Few rows in much padding: as many CTAs as its zeros keep busy.
  void widen_for_padding(Split* split, int ctas_per_sm) const {
    if (!t.offsets) return;
    const int64_t most = (int64_t)sm_count() * ctas_per_sm;
    split->grid = (unsigned)std::max<int64_t>(split->grid, std::min(most, ceil_div((int64_t)t.n_segments * t.L_max, 64)));
  }
  template <typename T, int KIND, int E, int TEAM, int V>
  int rows() const {
    constexpr int threads = norm::kCtaThreads<TEAM>, per_sm = norm::kBackwardThreads<KIND, E, TEAM, V>;
    constexpr int fixed = norm::kBackwardBytes<T, KIND, E, TEAM, V>;
    auto kern = norm::backward_rows_kernel<T, KIND, E, TEAM, V>;
    static std::atomic<unsigned char> configured[kMaxDevices];
    constexpr int most = fixed + (KIND == norm::kLayer ? norm::Wide<E>::bytes(TEAM * V * E) : 0);
    static_assert(most <= 227 * 1024, "shared memory of a CTA");
    static_assert(KIND != norm::kLayer || per_sm / threads <= norm::kSumCtas, "a row of the workspace for each CTA");
    if (int rc = ensure_smem(kern, most, configured)) return rc;
    // Unit rows that fill the 16 elements of every lane keep enough in flight with two CTAs on an SM instead
    // of three (781k x 128 bf16 93 and 104 us, 391k x 256 93 and 104; fp32 391k x 128, 195k x 256 and 98k x 512 98
    // and 100 each); rows that fill them in part do not (1042k x 96 bf16: 108 and 97).
    const bool full = KIND == norm::kUnit && V * E == 16 && t.dim == TEAM * V * E;
    const int ctas = full ? std::min(512, per_sm) / threads : per_sm / threads;
    Split split = share_rows<threads, TEAM>(std::max(t.rows, 1), ctas);
    widen_for_padding(&split, ctas);
    if (int rc = take_slabs(split.grid)) return rc;
    const int smem = fixed + (KIND == norm::kLayer ? norm::Wide<E>::bytes(t.dim) : 0);
    kern<<<split.grid, threads, smem, st>>>((const T*)grad, (const T*)tokens, split.of(t), weight, mean, rstd,
                                            (T*)grad_tokens, partial, eps);
    return launch_check("norm backward_rows_kernel");
  }
  template <typename T, int KIND, int E, int THREADS>
  int wide_rows(int ctas_per_sm) const {
    Split split = share_rows<THREADS, THREADS>(std::max(t.rows, 1), ctas_per_sm);
    widen_for_padding(&split, ctas_per_sm);
    norm::backward_wide_kernel<T, KIND, E, THREADS><<<split.grid, THREADS, 0, st>>>(
        (const T*)grad, (const T*)tokens, split.of(t), weight, mean, rstd, (T*)grad_tokens, eps);
    return launch_check("norm backward_wide_kernel");
  }
  template <typename T, int KIND, int E>
  int wide() const {
    if (grad_tokens) {
      const int rc = few_rows(t.rows) ? wide_rows<T, KIND, E, 1024>(1) : wide_rows<T, KIND, E, 256>(6);
      if (rc) return rc;
    }
    if (!partial) return MAXSIM_OK;
    if (int rc = take_slabs(std::min<int64_t>(grad_slabs(t.rows), 64))) return rc;
    norm::grad_weight_wide_kernel<T, E><<<dim3((unsigned)ceil_div(t.dim, norm::kThreads * E), (unsigned)slabs),
                                          norm::kThreads, 0, st>>>(
        (const T*)grad, (const T*)tokens, t, mean, rstd, partial, slabs);
    return launch_check("norm grad_weight_wide_kernel");
  }
};

template <typename W>
int launch_sum(const Backward& call, void* grad_weight, void* grad_bias) {
  norm::grad_weight_sum_kernel<W><<<dim3((unsigned)ceil_div(call.t.dim, 32), 2), norm::kSumThreads, 0, call.st>>>(
      call.partial, call.slabs, call.t.dim, (W*)grad_weight, (W*)grad_bias);
  return launch_check("norm grad_weight_sum_kernel");
}

}  // namespace
}  // namespace maxsim

using namespace maxsim;

extern "C" {

int64_t maxsim_b200_norm_rows_workspace(int64_t n_segments, int64_t L_max, int64_t dim) {
  if (n_segments <= 0 || L_max <= 0 || dim <= 0 || n_segments > kMaxRows / L_max) return 0;
  return workspace_bytes_for(grad_slabs(n_segments * L_max), dim);
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
  if (int rc = check_bases({grad, tokens, grad_tokens}, dtype, {weight, grad_weight, grad_bias}, weight_dtype)) return rc;
  if (n_segments * L_max == 0) {  // no rows: the sums are zero
    const size_t bytes = (size_t)dim * element_size(weight_dtype);
    if (grad_weight) MAXSIM_CUDA(cudaMemsetAsync(grad_weight, 0, bytes, st));
    if (grad_bias) MAXSIM_CUDA(cudaMemsetAsync(grad_bias, 0, bytes, st));
    return MAXSIM_OK;
  }
  if (!grad_tokens && !sums) return MAXSIM_OK;
  if (!tokens || (!grad && packed_rows > 0)) return fail(MAXSIM_EINVAL, "null pointer argument");
  if (kind == norm::kLayer && packed_rows > 0 && (!mean || !rstd)) return fail(MAXSIM_EINVAL, "null pointer argument");
  if (sums && (!workspace || workspace_bytes < maxsim_b200_norm_rows_workspace(n_segments, L_max, dim)))
    return fail(MAXSIM_EWORKSPACE, "workspace missing or smaller than maxsim_b200_norm_rows_workspace says");
  if (sums && (uintptr_t)workspace % sizeof(float) != 0)
    return fail(MAXSIM_EINVAL, "the workspace must start on a multiple of 4 bytes");
  const Backward call{grad, tokens, t, {weight, weight_dtype == MAXSIM_F32}, mean, rstd, grad_tokens,
                      sums ? static_cast<float*>(workspace) : nullptr, sums ? workspace_bytes : 0, (float)eps, st};
  if (int rc = launch(kind, dtype, call)) return rc;
  if (!sums) return MAXSIM_OK;
  switch (weight_dtype) {
    case MAXSIM_F32: return launch_sum<float>(call, grad_weight, grad_bias);
    case MAXSIM_F16: return launch_sum<__half>(call, grad_weight, grad_bias);
    default: return launch_sum<__nv_bfloat16>(call, grad_weight, grad_bias);
  }
}

}  // extern "C"
