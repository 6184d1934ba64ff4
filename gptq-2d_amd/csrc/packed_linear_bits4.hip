// The packed product's kernels for codes of 4 bits.
#include "packed_linear_kernels.h"

GPTQ2D_PACKED_PRODUCT(4) {
  return launch_mode<4>(*static_cast<const Linear*>(linear), *static_cast<const Plan*>(plan), st);
}
