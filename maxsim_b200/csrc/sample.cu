// extern "C" entry point of the sampling operator.
#include "host.h"
#include "sample.cuh"

namespace maxsim {
namespace {

template <int THREADS, bool CACHED>
int launch_rows(const sample::Args& A, cudaStream_t st) {
  auto kern = sample::sample_rows_kernel<THREADS, CACHED>;
  static std::atomic<unsigned char> configured[kMaxDevices];
  const size_t most = CACHED ? sample::kMostCached * sizeof(float) : 0;
  if (int rc = ensure_smem(kern, most, configured)) return rc;
  kern<<<(unsigned)A.rows, THREADS, CACHED ? (A.cols + 3) / 4 * 4 * sizeof(float) : 0, st>>>(A);
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
  if (cols <= 2048 && n <= 128 && rows > 4 * sms) return launch_rows<128, true>(A, st);
  if (cols <= 2048 || (cols <= 8192 && rows > 2 * sms)) return launch_rows<256, true>(A, st);
  if (cols <= 24576) return launch_rows<512, true>(A, st);
  if (cols <= sample::kMostCached) return launch_rows<1024, true>(A, st);
  return launch_rows<1024, false>(A, st);
}

}  // extern "C"
