// The norms before a branch with their result in 8 bits (gfx950), for the 8-bit
// linear layer after them: the kernels of modulate.h, which round the fp32 row where
// they would round it to bf16. Nothing but the row and its scales is written: 3 bytes
// a value against 7 for a bf16 row and its quantisation (7 against 11 with the
// residual). 6,240 x 5,376 with the residual: 48 to 50 us for 235 MB, 4.7 to 4.9 TB/s;
// 257 x 5,376 without: 3.6 us, two dependent rounds of loads and the row's sum.
#include "modulate.h"

namespace h3a {
namespace {

template <bool kResidual>
hipError_t launch_t(const ModulateParams& p, hipStream_t stream) {
    const int nv = (int)((p.cols + 8 * kThreads - 1) / (8 * kThreads));
    if (p.table_f32) {
        if (p.w_f32)
            launch_modulate_vec<kResidual, true, true, true>(p, nv, stream);
        else
            launch_modulate_vec<kResidual, true, false, true>(p, nv, stream);
    } else {
        if (p.w_f32)
            launch_modulate_vec<kResidual, false, true, true>(p, nv, stream);
        else
            launch_modulate_vec<kResidual, false, false, true>(p, nv, stream);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_modulate_fp8(const ModulateParams& p, hipStream_t stream) {
    if (p.rows == 0) return hipSuccess;
    return p.residual != nullptr ? launch_t<true>(p, stream) : launch_t<false>(p, stream);
}

}  // namespace h3a
