// How the kernels that copy rows of the pools (draft_cache.hip, score_evict.hip) choose
// the vector that one access moves.
#pragma once

#include "draft_cache.hpp"

#include <algorithm>

namespace mvr {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <typename F>
hipError_t with_vector(int64_t row_bytes, const void* a, const void* b, F launch) {
  const int bytes = cache_vector_bytes(row_bytes, a, b), row_vecs = (int)(row_bytes / bytes);
  if (bytes == 16) return launch(u32x4{}, row_vecs);
  if (bytes == 4) return launch(uint32_t{}, row_vecs);
  return launch(uint16_t{}, row_vecs);
}

} // namespace
} // namespace mvr
