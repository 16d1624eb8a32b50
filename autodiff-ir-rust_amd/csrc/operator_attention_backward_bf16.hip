// Backward kernels of attention for bf16.
#include "operator_attention_backward.hpp"

void adhip::attn::backward_bf16(const Params& p, hipStream_t stream) { backward<bf16>(p, stream); }
