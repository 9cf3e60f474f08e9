// The softmax loss's backward kernels for bfloat16 rows (softmax_tiles.h).
#define RECSDK_SOFTMAX_KERNELS
#include "softmax_tiles.h"

namespace recsdk {

int launch_bf16_backward(int pass, const LossArgs& a, const PassPlan& p, hipStream_t stream)
{
    return pass == kLossDx ? launch_pass<1, kLossDx>(a, p, stream) : launch_pass<1, kLossDt>(a, p, stream);
}

}  // namespace recsdk
