// The products of bf16 operands.
#include "product_type.cuh"

namespace mlpk {
namespace product {

int launch_bf16(const Product& p, cudaStream_t st) { return launch_type<__nv_bfloat16>(p, st); }

}  // namespace product
}  // namespace mlpk
