// extern "C" entry point of the sampling operator.
#include "host.h"
#include "sample.cuh"

namespace maxsim {
namespace {

template <int THREADS, bool CACHED>
int launch_rows(const sample::Args& A, cudaStream_t st) {
  auto kern = sample::sample_rows_kernel<THREADS, CACHED, false>;
  static std::atomic<unsigned char> configured[kMaxDevices];
  const size_t most = CACHED ? sample::kMostCached * sizeof(float) : 0;
  if (int rc = ensure_smem(kern, most, configured)) return rc;
  kern<<<(unsigned)A.rows, THREADS, CACHED ? (A.cols + 3) / 4 * 4 * sizeof(float) : 0, st>>>(A);
  return launch_check("sample_rows_kernel");
}

// The CTAs a row is split over, 0 for none: few rows that are long.  A cluster's barriers cost
// about 10 us a row, and clusters of 8 find room beside each other on three quarters of the SMs.  Measured,
// us without a filter / top-p / top-k, one row: of 12288 14 / 27 / 15 on one CTA and 14 / 24 / 17 on four;
// 16384 17 / 33 / 17 and 15 / 25 / 18; 40960 29 / 56 / 23, on four 19 / 38 / 21, on eight 17 / 35 / 20; 262144
// 256 / 524 / 101 and on eight 34 / 86 / 31; 2^20 983 / 2032 / 353, on eight 147 / 308 / 68, on 16 88 / 201 / 51.  18 rows of
// 70000 on four 26 / 49 / 26 and on eight (144 CTAs) 26 / 53 / 26; 74 rows of 40000 on one 29 / 56 / 24, on two 25 / 45 / 25.
int cluster_ctas(int64_t rows, int64_t cols, int sms) {
  const int64_t room = (int64_t)sms * 3 / 4;
  if (cols < 16384) return 0;
  if (cols > 8 * sample::kMostCached && rows * 16 <= room) return 16;
  if (cols > 32768 && rows * 8 <= room) return 8;
  if (rows * 4 <= room) return 4;
  return rows * 2 <= sms ? 2 : 0;
}

// A cluster of `ctas` CTAs per row.
template <int THREADS, bool CACHED>
int launch_clusters(const sample::Args& A, int ctas, cudaStream_t st) {
  auto kern = sample::sample_rows_kernel<THREADS, CACHED, true>;
  static std::atomic<unsigned char> configured[kMaxDevices];
  const size_t most = CACHED ? sample::kMostCached * sizeof(float) : 0;
  if (int rc = ensure_smem(kern, most, configured)) return rc;
  const int quads = (A.cols + 3) / 4, slice = (quads + ctas - 1) / ctas;
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)ctas;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(A.rows * ctas));
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = CACHED ? slice * 4 * sizeof(float) : 0;
  config.stream = st;
  config.attrs = &cluster;
  config.numAttrs = 1;
  if (ctas > 8) {  // not every device has room for that many side by side
    int fit = 0;
    MAXSIM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    MAXSIM_CUDA(cudaOccupancyMaxActiveClusters(&fit, kern, &config));
    if (fit < 1) return launch_clusters<1024, false>(A, 8, st);
  }
  MAXSIM_CUDA(cudaLaunchKernelEx(&config, kern, A));
  return launch_check("sample_rows_kernel");
}

}  // namespace
}  // namespace maxsim

using namespace maxsim;

extern "C" {

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
  if (A.shift > 51) A.shift = 51;
  A.indices = indices;
  A.probabilities = probabilities;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Threads of a row.  A CTA's barriers and reductions cost the same for few elements as for many:
  // with more rows than run at once small CTAs get more done, with fewer the row itself has to be quick.
  // Measured, top-p draws, us with 128 / 256 / 512 threads: 1 x 1000 10.4 / 9.4 / 10.2, 700 x 500 24.6 / 28.9 / 37.9;
  // 140 x 8000 29.5 / 20.3 / 16.6, 600 x 8000 56.7 / 42.3 / 47.5; 512 x 20000, where shared memory holds two
  // rows whatever their threads, 123 / 82 / 68.
  const int sms = sm_count();
  if (const int ctas = cluster_ctas(rows, cols, sms)) {
    if (cols > ctas * (int64_t)sample::kMostCached) return launch_clusters<1024, false>(A, ctas, st);
    // Threads: 400k in 16 slices 94 us with 512 and 103 with 1024, 70k in eight 40 and 43, 20k in two 32 and 32,
    // 40960 in two 53 and 44; slices that stay in memory, 2^20 in 16, 255 and 201.
    if (ctas > 8 || cols <= ctas * 11264) return launch_clusters<512, true>(A, ctas, st);
    return launch_clusters<1024, true>(A, ctas, st);
  }
  if (cols <= 2048 && n <= 128 && rows > 4 * sms) return launch_rows<128, true>(A, st);
  if (cols <= 2048 || (cols <= 8192 && rows > 2 * sms)) return launch_rows<256, true>(A, st);
  if (cols <= 24576) return launch_rows<512, true>(A, st);
  if (cols <= sample::kMostCached) return launch_rows<1024, true>(A, st);
  return launch_rows<1024, false>(A, st);
}

}  // extern "C"
