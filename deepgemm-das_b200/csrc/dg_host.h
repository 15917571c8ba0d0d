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

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace host
}  // namespace dg
