// Forward kernels of attention for bf16.
#include "operator_attention_forward.hpp"

void adhip::attn::forward_bf16(const Params& p, bool few_rows, hipStream_t stream) {
    switch (padded_size(p.D)) {
        case 32: return launch_forward<bf16, bf16, 32>(p, few_rows, stream);
        case 64: return launch_forward<bf16, bf16, 64>(p, few_rows, stream);
        case 96: return launch_forward<bf16, bf16, 96>(p, few_rows, stream);
        case 128: return launch_forward<bf16, bf16, 128>(p, few_rows, stream);
        case 192: return launch_forward<bf16, bf16, 192>(p, few_rows, stream);
        case 256: return launch_forward<bf16, bf16, 256>(p, few_rows, stream);
    }
}
