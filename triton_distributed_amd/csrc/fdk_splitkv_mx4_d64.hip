// Split-KV kernels over MXFP4 caches for head_dim = 64.
#include "fdk_splitkv_mx4.h"

namespace fdk {

int launch_splitkv_mx4_d64(const SplitParams& p, const Mx4Scales& x, int q_dtype, hipStream_t stream) {
    return q_dtype == FDK_BF16 ? launch_mx4<FDK_BF16, 64>(p, x, stream) : launch_mx4<FDK_FP16, 64>(p, x, stream);
}

}  // namespace fdk
