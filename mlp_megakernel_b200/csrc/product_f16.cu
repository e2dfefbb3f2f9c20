// The products of f16 operands.
#include "product_type.cuh"

namespace mlpk {
namespace product {

int launch_f16(const Product& p, cudaStream_t st) { return launch_type<__half>(p, st); }

}  // namespace product
}  // namespace mlpk
