// The packed product's kernels for codes of 8 bits.
#include "packed_linear_kernels.h"

GPTQ2D_PACKED_PRODUCT(8) {
  return launch_mode<8>(*static_cast<const Linear*>(linear), *static_cast<const Plan*>(plan), st);
}
