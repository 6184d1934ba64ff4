// The packed product's kernels for codes of 3 bits.
#include "packed_linear_kernels.h"

GPTQ2D_PACKED_PRODUCT(3) {
  return launch_mode<3>(*static_cast<const Linear*>(linear), *static_cast<const Plan*>(plan), st);
}
