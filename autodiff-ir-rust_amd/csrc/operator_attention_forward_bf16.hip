// Forward kernels of attention for bf16.
#include "operator_attention_forward.hpp"

void adhip::attn::forward_bf16(const Params& p, bool few_rows, hipStream_t stream) { forward<bf16>(p, few_rows, stream); }
