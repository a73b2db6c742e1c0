// Shared by the operators that work on tensors of three types (fp32, bf16, fp16): type codes, matrix-core fragments, argument structs.
#pragma once
#include "common.hpp"

namespace icap {

enum DType : int { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Vec;
template <> struct Vec<float> { typedef f32x8 x8; typedef f32x4 x4; };
template <> struct Vec<__bf16> { typedef bf16x8 x8; typedef bf16x4 x4; };
template <> struct Vec<_Float16> { typedef f16x8 x8; typedef f16x4 x4; };

struct AttnArgs {
    const void *q, *k, *v, *dout, *o;       // element strides below; o dense [tokens_q][heads][dim]
    void *out, *dq, *dk, *dv;               // dense
    float *lse, *delta, *part;              // lse, delta [tokens_q][heads]; part: partial results of split keys
    const int *cu_q, *cu_k;
    int seqs, tokens_q, tokens_k, heads, kv_heads, group, dim, causal, splits;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head, g_tok, g_head;
    float scale;
};

int attention_fwd_f32(const AttnArgs&, hipStream_t);
int attention_fwd_bf16(const AttnArgs&, hipStream_t);
int attention_fwd_f16(const AttnArgs&, hipStream_t);
int attention_bwd_f32(const AttnArgs&, hipStream_t);
int attention_bwd_bf16(const AttnArgs&, hipStream_t);
int attention_bwd_f16(const AttnArgs&, hipStream_t);

}  // namespace icap
