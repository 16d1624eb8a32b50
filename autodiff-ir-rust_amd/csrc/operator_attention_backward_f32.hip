// Backward kernels of attention for f32, up to 128 features.
#include "operator_attention_backward.hpp"

void adhip::attn::backward_f32(const Params& p, hipStream_t stream) {
    switch (padded_size(p.D)) {
        case 32: return launch_backward<Parts, 32>(p, stream);
        case 64: return launch_backward<Parts, 64>(p, stream);
        case 96: return launch_backward<Parts, 96>(p, stream);
        case 128: return launch_backward<Parts, 128>(p, stream);
        default: return backward_f32_wide(p, stream);
    }
}
