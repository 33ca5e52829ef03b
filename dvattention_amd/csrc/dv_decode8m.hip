// Attention over 8-bit caches, row groups of four tokens, fp32 of two (kernels:
// dv_decode8.h).  Built with accumulators in AGPRs.
#include "dv_decode8.h"

namespace dv {

hipError_t launch_decode8_wide(int dtype, bool varlen, const DecodeParams& p, int device, long long cap, int cus,
                               hipStream_t stream) {
    if (dtype == kF32)
        return varlen ? launch8_one<kF32, kQRotHalf, kRowVarlen, 2, true, true>(p, device, cap, cus, stream)
                      : launch8_one<kF32, kQRotFull, kRowWS, 2, true, true>(p, device, cap, cus, stream);
    if (varlen) return hipErrorInvalidValue;
    if (dtype == kBF16) return launch8_one<kBF16, kQRotFull, kRowWS, 4, true, true>(p, device, cap, cus, stream);
    if (dtype == kF16) return launch8_one<kF16, kQRotFull, kRowWS, 4, true, true>(p, device, cap, cus, stream);
    return hipErrorInvalidValue;
}

}  // namespace dv
