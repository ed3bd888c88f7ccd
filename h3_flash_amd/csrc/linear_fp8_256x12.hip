// Tile kernels of the 8-bit linear layers: shapes of 256 features x 192 tokens.
#include "linear_fp8_tile.h"

namespace h3a {

template hipError_t launch_linear_fp8_tile<256, 12, 3, 2>(const LinearFp8Params&, hipStream_t);

}  // namespace h3a
