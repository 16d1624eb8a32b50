// Forward kernels of attention for f32.
#include "operator_attention_forward.hpp"

void adhip::attn::forward_f32(const Params& p, bool few_rows, hipStream_t stream) { forward<float>(p, few_rows, stream); }
