// The softmax loss's forward kernels for bfloat16 rows (softmax_tiles.h).
#define RECSDK_SOFTMAX_KERNELS
#include "softmax_tiles.h"

namespace recsdk {

int launch_bf16_forward(const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    return launch_pass<1, kLossForward>(a, p, stream);
}

}  // namespace recsdk
