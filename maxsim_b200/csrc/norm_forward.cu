// extern "C" entry point of the row normalisation operators.
#include "norm_host.cuh"

namespace maxsim {
namespace {

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
    constexpr int ring = norm::kRingBytes<T, E, TEAM, V, 1>;
    auto kern = norm::forward_rows_kernel<T, KIND, E, TEAM, V>;
    static std::atomic<unsigned char> configured[kMaxDevices];
    constexpr int most = ring + (KIND == norm::kLayer ? 2 * norm::Wide<E>::bytes(TEAM * V * E) : 0);
    static_assert(most <= 227 * 1024, "shared memory of a CTA");
    if (int rc = ensure_smem(kern, most, configured)) return rc;
    // Layer norms of floats with many packs: one CTA of 256 threads on an SM moves more than two
    // (130k x 768 139 and 131 us, 24k x 4096 160 and 151).
    constexpr int on_sm = KIND == norm::kLayer && E == 4 && V * E > 16 ? 256 : per_sm;
    const Split split = share_rows<threads, TEAM>(t.rows, on_sm / threads);
    const int smem = ring + (KIND == norm::kLayer ? 2 * norm::Wide<E>::bytes(t.dim) : 0);
    kern<<<split.grid, threads, smem, st>>>((const T*)tokens, split.of(t), weight, bias, (T*)out, mean, rstd, eps);
    return launch_check(name());
  }
  template <typename T, int KIND, int E, int THREADS>
  int wide_rows(int ctas_per_sm) const {
    const Split split = share_rows<THREADS, THREADS>(t.rows, ctas_per_sm);
    norm::forward_wide_kernel<T, KIND, E, THREADS><<<split.grid, THREADS, 0, st>>>(
        (const T*)tokens, split.of(t), weight, bias, (T*)out, mean, rstd, eps);
    return launch_check("norm forward_wide_kernel");
  }
  template <typename T, int KIND, int E>
  int wide() const {
    return few_rows(t.rows) ? wide_rows<T, KIND, E, 1024>(1) : wide_rows<T, KIND, E, 256>(6);
  }
};

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
  if (int rc = check_bases({tokens, out}, dtype, {weight, bias}, weight_dtype)) return rc;
  if (t.rows == 0) return MAXSIM_OK;
  if (!tokens || !out) return fail(MAXSIM_EINVAL, "null pointer argument");
  if ((mean == nullptr) != (rstd == nullptr)) return fail(MAXSIM_EINVAL, "mean and rstd come together");
  if (kind == norm::kUnit && (weight || bias)) return fail(MAXSIM_EINVAL, "unit rows have no weights");
  const bool f32 = weight_dtype == MAXSIM_F32;
  return launch(kind, dtype, Forward{tokens, t, {weight, f32}, {bias, f32}, out, mean, rstd, (float)eps,
                                     static_cast<cudaStream_t>(stream)});
}

int maxsim_b200_pack_norm_rows(int kind, const void* padded, int64_t segment_stride, int64_t row_stride,
                               const int32_t* lengths, int32_t* offsets, const void* weight, const void* bias,
                               void* packed, float* mean, float* rstd, int64_t n_segments, int64_t L_max,
                               int64_t dim, int64_t packed_rows, double eps, int dtype, int weight_dtype,
                               void* stream) {
  if (!offsets) return fail(MAXSIM_EINVAL, "null pointer argument");
  norm::Rows t;  // refuse before anything is written
  if (int rc = check_rows(kind, n_segments, L_max, dim, packed_rows, segment_stride, row_stride, offsets, eps, &t))
    return rc;
  if (int rc = maxsim_b200_offsets_from_lengths(lengths, n_segments, L_max, offsets, nullptr, stream)) return rc;
  return maxsim_b200_norm_rows(kind, padded, segment_stride, row_stride, offsets, weight, bias, packed, mean, rstd,
                               n_segments, L_max, dim, packed_rows, eps, dtype, weight_dtype, stream);
}

}  // extern "C"
