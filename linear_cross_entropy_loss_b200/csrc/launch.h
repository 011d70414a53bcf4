// What the translation units of the library share on the host side.
#pragma once

#include "../../include/lce_b200.h"

#include <cuda_runtime.h>
#include <atomic>

namespace lce {

// Kernels launched by the library in this process (lce_launch_count); defined in lce_api.cu.
extern std::atomic<long long> g_launches;

inline int check_launch() {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return cudaGetLastError() == cudaSuccess ? LCE_OK : LCE_ERR_CUDA;
}

}  // namespace lce
