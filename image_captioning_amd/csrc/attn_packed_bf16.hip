// Attention over packed sequences for bf16 tensors (the kernels: attn_packed.hpp).
#include "attn_packed.hpp"

namespace icap {

int attention_fwd_bf16(const AttnArgs& a, hipStream_t st) { return attn::fwd<__bf16>(a, st); }
int attention_bwd_bf16(const AttnArgs& a, hipStream_t st) { return attn::bwd<__bf16>(a, st); }

}  // namespace icap
