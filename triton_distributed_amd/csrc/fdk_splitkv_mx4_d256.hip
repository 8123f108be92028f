// Split-KV kernels over MXFP4 caches for head_dim = 256.
#include "fdk_splitkv_mx4.h"

namespace fdk {

int launch_splitkv_mx4_d256(const SplitParams& p, const Mx4Scales& x, int q_dtype, hipStream_t stream) {
    return q_dtype == FDK_BF16 ? launch_mx4<FDK_BF16, 256>(p, x, stream) : launch_mx4<FDK_FP16, 256>(p, x, stream);
}

}  // namespace fdk
