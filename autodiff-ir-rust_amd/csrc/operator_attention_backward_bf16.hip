// Backward kernels of attention for bf16.
#include "operator_attention_backward.hpp"

void adhip::attn::backward_bf16(const Params& p, hipStream_t stream) {
    switch (padded_size(p.D)) {
        case 32: return launch_backward<bf16, 32>(p, stream);
        case 64: return launch_backward<bf16, 64>(p, stream);
        case 96: return launch_backward<bf16, 96>(p, stream);
        case 128: return launch_backward<bf16, 128>(p, stream);
        case 192: return launch_backward<bf16, 192>(p, stream);
        case 256: return launch_backward<bf16, 256>(p, stream);
    }
}
