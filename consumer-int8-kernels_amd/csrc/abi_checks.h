// Argument checks and status reporting shared by the C entry points (abi.cpp,
// attention_abi.cpp). Host code only.
#pragma once
#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace ci8 {

// Stores the calling thread's message for ci8_last_error() and returns `status`.
int abi_fail(int status, const char* message);
// CI8_OK and an empty message, or CI8_ERR_LAUNCH with the runtime's.
int abi_launched(hipError_t error);

inline bool aligned(const void* p, uintptr_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

inline bool overlap(const void* a, int64_t bytes_a, const void* b, int64_t bytes_b) {
  const auto first = reinterpret_cast<uintptr_t>(a);
  const auto second = reinterpret_cast<uintptr_t>(b);
  return bytes_a > 0 && bytes_b > 0 && first < second + uint64_t(bytes_b) &&
         second < first + uint64_t(bytes_a);
}

inline hipStream_t as_stream(void* stream) { return static_cast<hipStream_t>(stream); }

}  // namespace ci8
