// What stands behind a product in its epilogue (product_kernel.cuh).
#pragma once

namespace mlpk {

enum Epi : int { kEpiPlain, kEpiLinear, kEpiGated, kEpiGatedBwd };

}  // namespace mlpk
