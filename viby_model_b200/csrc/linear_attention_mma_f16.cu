// Tensor-core linear attention, fp16.
#include "linear_attention_mma.cuh"

namespace vc1d {
cudaError_t launch_linear_mma_f16(const lin::Launch& l, bool states_only, cudaStream_t s) {
    return lin::mma::launch_type<VC1D_F16>(l, states_only, s);
}
}  // namespace vc1d
