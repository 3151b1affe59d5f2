// Linear attention on the fifth-generation tensor cores: bf16.
#include "linear_attention_tc.cuh"

namespace vc1d {

cudaError_t launch_linear_tc(const lin::Launch& l, bool states_only, cudaStream_t s) {
    unsigned int* timeouts = tma::timeouts_ptr();
    if (timeouts == nullptr) return cudaErrorNotSupported;
    const int da = lin::largest_rows(l);
    const bool rev = l.run[0].reverse != 0;  // the runs of a launch go the same way
    if (da <= 128)
        return states_only ? (rev ? lin::tc::launch<128, true, true>(l, timeouts, s) : lin::tc::launch<128, true, false>(l, timeouts, s))
                           : (rev ? lin::tc::launch<128, false, true>(l, timeouts, s) : lin::tc::launch<128, false, false>(l, timeouts, s));
    return states_only ? (rev ? lin::tc::launch<160, true, true>(l, timeouts, s) : lin::tc::launch<160, true, false>(l, timeouts, s))
                       : (rev ? lin::tc::launch<160, false, true>(l, timeouts, s) : lin::tc::launch<160, false, false>(l, timeouts, s));
}

}  // namespace vc1d
