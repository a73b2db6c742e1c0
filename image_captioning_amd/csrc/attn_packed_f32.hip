// Attention over packed sequences for fp32 tensors (the kernels: attn_packed.hpp).
#include "attn_packed.hpp"

namespace icap {

int attention_fwd_f32(const AttnArgs& a, hipStream_t st) { return attn::fwd<float>(a, st); }
int attention_bwd_f32(const AttnArgs& a, hipStream_t st) { return attn::bwd<float>(a, st); }

}  // namespace icap
