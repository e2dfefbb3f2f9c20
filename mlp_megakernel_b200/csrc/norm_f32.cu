// The RMS norm's kernels for fp32 rows.
#include "norm_launch.cuh"

namespace mlpk {
namespace norm {
int forward_f32(const NormArgs& a, bool w32, bool fp8, cudaStream_t st) {
  return forward_of<float>(a, w32, fp8, st);
}
int backward_f32(const NormBwdArgs& a, bool w32, int64_t blocks, void* dw, int dev, cudaStream_t st) {
  return backward_of<float>(a, w32, blocks, dw, dev, st);
}
}  // namespace norm
}  // namespace mlpk
