// Backward kernels of attention for f32.
#include "operator_attention_backward.hpp"

void adhip::attn::backward_f32(const Params& p, hipStream_t stream) { backward<float>(p, stream); }
