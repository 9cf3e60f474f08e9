// The softmax loss's forward kernels for float32 rows (softmax_tiles.h).
#define RECSDK_SOFTMAX_KERNELS
#include "softmax_tiles.h"

namespace recsdk {

int launch_f32_forward(int planes, const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    return planes == 2 ? launch_pass<2, kLossForward>(a, p, stream) : launch_pass<3, kLossForward>(a, p, stream);
}

}  // namespace recsdk
