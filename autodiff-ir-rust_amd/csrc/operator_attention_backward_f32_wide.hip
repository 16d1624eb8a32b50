// Backward kernels of attention for f32, 129 to 256 features: three planes of parts would fit neither registers nor LDS, so
// these run on the FP32 matrix cores.
#include "operator_attention_backward.hpp"

void adhip::attn::backward_f32_wide(const Params& p, hipStream_t stream) {
    if (padded_size(p.D) == 192) launch_backward<float, 192>(p, stream);
    else launch_backward<float, 256>(p, stream);
}
