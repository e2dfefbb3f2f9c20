// The products of f16 operands.
#include "product_type.cuh"

namespace mlpk {
namespace product {

int64_t workspace_bytes(const Product& p, int sm_count) {  // the same for both types
  if (few_rows(p, sm_count)) return 0;
  return plan_of(p, sm_count / 2).partials() * static_cast<int64_t>(sizeof(float));
}

int launch_f16(const Product& p, cudaStream_t st) { return launch_type<__half>(p, st); }

}  // namespace product
}  // namespace mlpk
