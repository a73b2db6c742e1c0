// Attention over packed sequences for fp16 tensors (the kernels: attn_packed.hpp).
#include "attn_packed.hpp"

namespace icap {

int attention_fwd_f16(const AttnArgs& a, hipStream_t st) { return attn::fwd<_Float16>(a, st); }
int attention_bwd_f16(const AttnArgs& a, hipStream_t st) { return attn::bwd<_Float16>(a, st); }

}  // namespace icap
