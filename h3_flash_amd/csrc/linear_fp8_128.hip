// Tile kernels of the 8-bit linear layers: shapes of 128 features.
#include "linear_fp8_tile.h"

namespace h3a {

template hipError_t launch_linear_fp8_tile<128, 8, 5, 4>(const LinearFp8Params&, hipStream_t);
template hipError_t launch_linear_fp8_tile<128, 6, 6, 4>(const LinearFp8Params&, hipStream_t);
template hipError_t launch_linear_fp8_tile<128, 4, 6, 5>(const LinearFp8Params&, hipStream_t);
template hipError_t launch_linear_fp8_tile<128, 2, 8, 6>(const LinearFp8Params&, hipStream_t);

}  // namespace h3a
