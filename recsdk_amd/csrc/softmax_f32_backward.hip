// The softmax loss's backward kernels for float32 rows (softmax_tiles.h).
#define RECSDK_SOFTMAX_KERNELS
#include "softmax_tiles.h"

namespace recsdk {

int launch_f32_backward(int pass, int planes, const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    if (pass == kLossDx) {
        return planes == 2 ? launch_pass<2, kLossDx>(a, p, stream) : launch_pass<3, kLossDx>(a, p, stream);
    }
    return planes == 2 ? launch_pass<2, kLossDt>(a, p, stream) : launch_pass<3, kLossDt>(a, p, stream);
}

}  // namespace recsdk
