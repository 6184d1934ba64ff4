// The packed product's kernels for codes of 2 bits.
#include "packed_linear_kernels.h"

GPTQ2D_PACKED_PRODUCT(2) {
  return launch_mode<2>(*static_cast<const Linear*>(linear), *static_cast<const Plan*>(plan), st);
}
