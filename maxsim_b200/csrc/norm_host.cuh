// Host side of the row normalisation operators, shared by the forward and the
// backward translation unit: argument checks, the split of the rows over a grid and the
// choice of a kernel.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>

#include "host.h"
#include "norm.cuh"

namespace maxsim {
namespace {

constexpr int64_t kMaxRows = (1ll << 31) - 4096;  // 32-bit row counters run a few turns ahead

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How the packed rows are split over a grid: every CTA gets the same number of
// consecutive rows, whole turns of its teams.
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
  constexpr int together = THREADS / TEAM;
  const int64_t most = (int64_t)sm_count() * ctas_per_sm;
  const int64_t chunk = ceil_div(ceil_div(rows, most), together) * together;
  return {(unsigned)ceil_div(rows, chunk), (int32_t)chunk};
}

// Rows of more than 4096 elements: as few as this get a CTA that fills an SM.
bool few_rows(int64_t rows) { return rows <= 2 * sm_count(); }

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
  return call.template wide<T, KIND, E>();
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

int check_types(int dtype, int weight_dtype) {
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype)) return fail(MAXSIM_EINVAL, "unknown dtype code");
  if (weight_dtype != dtype && weight_dtype != MAXSIM_F32)
    return fail(MAXSIM_EUNSUPPORTED, "weights must be float or of the tokens' type");
  return MAXSIM_OK;
}

int element_size(int dtype) { return dtype == MAXSIM_F32 ? 4 : 2; }

// Every pointer on a multiple of its element's size.
int check_bases(std::initializer_list<const void*> rows, int dtype, std::initializer_list<const void*> weights,
                int weight_dtype) {
  bool bad = false;
  for (const void* p : rows) bad |= (uintptr_t)p % element_size(dtype) != 0;
  for (const void* p : weights) bad |= (uintptr_t)p % element_size(weight_dtype) != 0;
  return bad ? fail(MAXSIM_EINVAL, "a base address is not a multiple of its element size") : MAXSIM_OK;
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
