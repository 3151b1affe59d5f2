// Linear attention on the fifth-generation tensor cores: bf16.
#include "linear_attention_tc.cuh"

namespace vc1d {

cudaError_t launch_linear_tc(const lin::Launch& l, bool states_only, cudaStream_t s) {
    unsigned int* timeouts = tma::timeouts_ptr();
    if (timeouts == nullptr) return cudaErrorNotSupported;
    int da = 0;
    for (int i = 0; i < l.runs; ++i) da = max(da, l.run[i].da);
    if (da <= 128) return states_only ? lin::tc::launch<128, true>(l, timeouts, s) : lin::tc::launch<128, false>(l, timeouts, s);
    return states_only ? lin::tc::launch<160, true>(l, timeouts, s) : lin::tc::launch<160, false>(l, timeouts, s);
}

}  // namespace vc1d
