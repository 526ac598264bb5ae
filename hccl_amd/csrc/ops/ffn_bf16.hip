// The experts' feed-forward kernels for bf16.
#include "hccl_types.h"
#include "ops/ffn_launch.h"

namespace hcclx {
template hipError_t launch_ffn<HCCL_DATA_TYPE_BFP16>(FfnKind, const FfnArgs &, uint32_t, hipStream_t);
}  // namespace hcclx
