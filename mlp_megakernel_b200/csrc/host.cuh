// Host-side helpers shared by the library's translation units: device
// look-up, launch through cudaLaunchKernelEx, and the record of the calling
// thread's last CUDA failure.  The functions are defined in mlpk_api.cu and
// are not exported.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <utility>

#include "../../include/mlpk.h"

namespace mlpk {
namespace host {

struct DevInfo {
  int sm_count = 0;
  int major = 0;
  int minor = 0;
  bool valid = false;
};

// MLPK_OK, or MLPK_ERR_CUDA with the failure kept for mlpk_last_cuda_error.
__attribute__((visibility("hidden"))) int cuda_status(cudaError_t e);

// The current device's properties; MLPK_ERR_ARCH if it is not sm_100.
__attribute__((visibility("hidden"))) int current_device_info(DevInfo* out, int* dev_out);

constexpr int kMaxBlockSmem = 227 * 1024;  // dynamic shared memory of a block

// Blocks of a kernel that an SM holds at a time (found once for each size; also
// lets the kernel have that much dynamic shared memory); 0 on a failure, whose
// status is kept for mlpk_last_cuda_error.
__attribute__((visibility("hidden"))) int blocks_per_sm(const void* kern, int threads, size_t smem, int dev);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch through cudaLaunchKernelEx so that the status returned is that of
// THIS launch, not an error left earlier on the calling thread.  With `early`
// the kernel is launched with programmatic stream serialization: it may start
// while the kernel before it on the stream is still running (every kernel of
// the library calls pdl_enter() before touching global memory, ptx.cuh), so
// its setup overlaps that kernel's tail.  The inference forward launches this
// way (back-to-back small calls: 6.0 -> 5.2 us per call at 64 rows); the
// training kernels do not (the config-3 step measured 40.8 us at 16,384 rows
// without it, 42.4 with it).
template <typename... KArgs, typename... Args>
int launch_kernel_cfg(bool early, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                      cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...));
}
template <typename... KArgs, typename... Args>
int launch_kernel(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                  Args&&... args) {
  return launch_kernel_cfg(false, kern, grid, block, smem, st, std::forward<Args>(args)...);
}
template <typename... KArgs, typename... Args>
int launch_kernel_early(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                        Args&&... args) {
  return launch_kernel_cfg(true, kern, grid, block, smem, st, std::forward<Args>(args)...);
}

}  // namespace host
}  // namespace mlpk
