// What the C entry points of several files share: the calling thread's error
// text, checked mode, trace ranges and the scalar checks of attention
// arguments.  Defined in mvr_attn_api.cpp.
#pragma once

#include "mvr_attn.h"

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <exception>
#include <vector>

namespace mvr {
namespace api {

// Sets the thread's error text and returns code.
__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...);
void clear_error();

// MVR_ATTN_CHECKED=true: calls check their device tables on the host first.
bool checked();

// A positive integer from the environment.
int env_int(const char* name, int fallback);

// Host copy of `count` int32 device values (none when dev is null), after
// waiting for the stream; false if the copy fails.
bool copy_to_host(const int32_t* dev, size_t count, void* stream, std::vector<int32_t>& host);

// mvr_paged_attention's checks of its scalar arguments.
int check_attention_scalars(const mvr_paged_attention_args* a);

// Compute units of the current device (256 where none can be asked).
int compute_units();

// A roctx range around a call, on when MVR_ENABLE_ROCTX=true.
class Range {
 public:
  explicit Range(const char* name);
  ~Range();

 private:
  bool on_;
};

// ---- for the entry points of the calls beside mvr_attn.h's own ----

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

inline int es_of(int32_t dtype) { return dtype == MVR_DTYPE_F16 ? 2 : 4; }

inline int launch_status(hipError_t err) {
  return err == hipSuccess ? MVR_OK : fail(MVR_E_HIP, "kernel launch failed: %s", hipGetErrorString(err));
}

inline const int32_t* data_or_null(const std::vector<int32_t>& v) { return v.empty() ? nullptr : v.data(); }

// Checked mode: runs `check` on host copies of the device tables; the host
// memory that they take may not be there.
template <typename F>
int run_checked(F check) {
  try {
    return check();
  } catch (const std::exception&) { // (bad_alloc, or more than a vector may hold)
    return fail(MVR_E_INVALID_ARGUMENT, "checked mode: out of host memory");
  }
}

// Threads of one launch, over all its blocks.
constexpr int64_t kMaxThreads = UINT32_MAX;

// Host tables of q_lens: starts that ascend from 0 and end by total_q (0: not given).
// Whatever is read per token afterwards lies within them.
inline int check_cu_q_lens(const int32_t* cu, int num_seqs, int32_t total_q, int32_t max_q_len = INT32_MAX) {
  if (cu[0] != 0) return fail(MVR_E_INVALID_ARGUMENT, "cu_q_lens[0] must be 0");
  for (int s = 0; s < num_seqs; s++)
    if (cu[s + 1] < cu[s] || (int64_t)cu[s + 1] - cu[s] > max_q_len)
      return max_q_len == INT32_MAX
                 ? fail(MVR_E_INVALID_ARGUMENT, "cu_q_lens decreases at request %d", s)
                 : fail(MVR_E_INVALID_ARGUMENT, "request %d has q_len %lld outside [0, max_q_len %d]", s,
                        (long long)cu[s + 1] - cu[s], max_q_len);
  if (total_q > 0 && cu[num_seqs] > total_q)
    return fail(MVR_E_INVALID_ARGUMENT, "cu_q_lens[num_seqs] = %d exceeds total_q = %d", cu[num_seqs], total_q);
  return MVR_OK;
}

inline int copy_failed() { return fail(MVR_E_HIP, "checked mode: copying the device tables to the host failed"); }

// Geometry and alignment of a call's K and V pools.
inline int check_pool(int32_t dtype, int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int64_t num_pages,
                      const void* key_pool, const void* value_pool) {
  if (dtype != MVR_DTYPE_F32 && dtype != MVR_DTYPE_F16)
    return fail(MVR_E_UNSUPPORTED, "dtype %d is not F32 (0) or F16 (1)", dtype);
  if (num_kv_heads < 1 || page_size < 1 || head_dim < 1 || num_pages < 1)
    return fail(MVR_E_INVALID_ARGUMENT, "invalid pool geometry");
  // A page's elements are counted in 32 bits.
  if ((int64_t)num_kv_heads * page_size > INT32_MAX / head_dim)
    return fail(MVR_E_UNSUPPORTED, "pages of 2^31 elements or more");
  if (!key_pool || !value_pool) return fail(MVR_E_INVALID_ARGUMENT, "null pool pointer");
  if (((uintptr_t)key_pool | (uintptr_t)value_pool) % es_of(dtype))
    return fail(MVR_E_INVALID_ARGUMENT, "pools must be aligned to their elements");
  return MVR_OK;
}

} // namespace api
} // namespace mvr
