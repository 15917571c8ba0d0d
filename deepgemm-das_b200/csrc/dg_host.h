// Host-side helpers shared by the translation units of the library (internal, not exported).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "deepgemm_b200.h"

namespace dg {
namespace host {

constexpr int kMaxDevices = 64;

struct DeviceInfo {
  std::once_flag once;
  int status = DG_ERR_NO_DEVICE;
  int sm_count = 0;
  int max_smem = 0;
  int cc = 0;
};

// Records the error for dg_last_cuda_error() and returns DG_ERR_CUDA.
int cuda_fail(cudaError_t e);

// Properties of the current device, read once; DG_OK if it is a device this library runs on.
int device_info(const DeviceInfo** out);

// rank-2 or rank-3 tiled map; dims / strides innermost first, strides in bytes for dims 1..
int encode_map(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base,
               const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
               CUtensorMapSwizzle swizzle);

// Adds to dg_query(DG_QUERY_LAUNCH_COUNT).
void count_launches(int n);

// Whether a buffer of `n` bytes and one of `m` share any: a result must not lie on what it is made of,
// which other blocks may still be reading.
inline bool overlap(const void* a, long long n, const void* b, long long m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a != nullptr && b != nullptr && n > 0 && m > 0 && (x < y ? y - x < static_cast<uintptr_t>(n) : x - y < static_cast<uintptr_t>(m));
}
// Bytes from the first to behind the last of `rows` rows of `h` elements, `stride` apart.
inline long long row_span(long long rows, long long stride, long long h, long long elem_bytes) {
  return rows > 0 ? ((rows - 1) * stride + h) * elem_bytes : 0;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace host
}  // namespace dg
