// Forward kernels of attention for f32.
#include "operator_attention_forward.hpp"

void adhip::attn::forward_f32(const Params& p, bool few_rows, hipStream_t stream) {
    switch (padded_size(p.D)) {
        case 32: return launch_forward<Parts, Split, 32>(p, few_rows, stream);
        case 64: return launch_forward<Parts, Split, 64>(p, few_rows, stream);
        case 96: return launch_forward<Parts, Split, 96>(p, few_rows, stream);
        case 128: return launch_forward<Parts, Split, 128>(p, few_rows, stream);
        case 192: return launch_forward<Split, Split, 192>(p, few_rows, stream);
        case 256: return launch_forward<Split, Split, 256>(p, few_rows, stream);
    }
}
