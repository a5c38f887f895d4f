// Shared host-side helpers of the C-ABI library: thread-local error text,
// CUDA error mapping, launch counting.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/mac_b200.h"

namespace mac_b200 {

// Text behind mac_b200_last_error(); one buffer per host thread.
char* error_buffer();
constexpr int kErrorBufferBytes = 512;

int fail(int code, const char* fmt, ...);

inline int cuda_fail(cudaError_t err, const char* what) {
  return fail(MAC_B200_ECUDA, "%s: %s (%s)", what, cudaGetErrorString(err),
              cudaGetErrorName(err));
}

// Where the sticky status bits of a file's kernels lie on the current device: the prefill ring build, its
// tensor-memory variant, the chunk attention, the 8-bit pool's kernels.  mac_b200_query_status takes them
// all in one exchange on the device.
int prefill_build_status_word(unsigned** word);
int prefill_sink_tc_status_word(unsigned** word);
int chunk_status_word(unsigned** word);
int kv8_status_word(unsigned** word);

// Sink-exclusive prefill build on tcgen05 / tensor memory (validated arguments); sets
// *launched when it ran, leaves it false when this step has to take the mma.sync kernel.
int launch_prefill_sink_exclusive_tc(const ::MacB200PrefillBuildArgs& a, int sms, cudaStream_t stream,
                                     bool* launched);

// Whether [a, a + a_bytes) and [b, b + b_bytes) have a byte in common.
inline bool byte_ranges_meet(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x <= y ? y - x < static_cast<uintptr_t>(a_bytes) : x - y < static_cast<uintptr_t>(b_bytes);
}

// Multiprocessor count of a device, looked up once per device.
int device_sm_count(int device);

// Kernels launched by this process through the library (all entry points).
extern std::atomic<int64_t> g_kernel_launches;

#define MAC_REQUIRE(cond, ...)                        \
  do {                                                \
    if (!(cond)) return ::mac_b200::fail(MAC_B200_EINVAL, __VA_ARGS__); \
  } while (0)

#define MAC_CUDA(call)                                              \
  do {                                                              \
    cudaError_t _e = (call);                                        \
    if (_e != cudaSuccess) return ::mac_b200::cuda_fail(_e, #call); \
  } while (0)

}  // namespace mac_b200
