// What the C entry points of several files share: the calling thread's error
// text, checked mode, trace ranges and the scalar checks of attention
// arguments.  Defined in mvr_attn_api.cpp.
#pragma once

#include "mvr_attn.h"

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

} // namespace api
} // namespace mvr
