// Tensor-core linear attention, bf16.
#include "linear_attention_mma.cuh"

namespace vc1d {
cudaError_t launch_linear_mma_bf16(const lin::Launch& l, bool states_only, cudaStream_t s) {
    return lin::mma::launch_type<VC1D_BF16>(l, states_only, s);
}
}  // namespace vc1d
