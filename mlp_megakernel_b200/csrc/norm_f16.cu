// The RMS norm's kernels for fp16 rows.
#include "norm_launch.cuh"

namespace mlpk {
namespace norm {
int forward_f16(const NormArgs& a, bool w32, bool fp8, cudaStream_t st) {
  return forward_of<__half>(a, w32, fp8, st);
}
int backward_f16(const NormBwdArgs& a, bool w32, int64_t blocks, void* dw, int dev, cudaStream_t st) {
  return backward_of<__half>(a, w32, blocks, dw, dev, st);
}
}  // namespace norm
}  // namespace mlpk
