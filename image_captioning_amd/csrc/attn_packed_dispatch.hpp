// Which attention kernel a call takes: the rows (for dK and dV the keys) of an average sequence decide.
//   up to 16: one wave a workgroup (single tokens fill their tile with the heads of a group; keys are split over workgroups)
//   16-bit: the 32-row waves of attn_packed_wide.hpp, as many as cover an average sequence, 2 to 8 (a workgroup shares each staged tile)
//   fp32: four waves of 16 rows
#pragma once
#include "attn_packed_wide.hpp"

namespace icap {
namespace attn {

template <typename T, int DP>
int fwd_dim(const AttnArgs& a, hipStream_t st) {
    const long long rows = (long long)a.tokens_q * a.group / a.seqs;
    if (rows <= 16) return launch_fwd<T, DP, 1, 1>(a, st);
    if constexpr (sizeof(T) == 4) return launch_fwd<T, DP, 4, 1>(a, st);
    else {
        if (rows <= 96) return launch_fwd_wide<T, DP, 2>(a, st);
        if (rows <= 512) return launch_fwd_wide<T, DP, 4>(a, st);
        return launch_fwd_wide<T, DP, 8>(a, st);
    }
}

template <typename T, int DP>
int bwd_dim(const AttnArgs& a, hipStream_t st) {
    const long long rows = (long long)a.tokens_q * a.group / a.seqs, keys = a.tokens_k / a.seqs;
    int rc;
    if (rows <= 16) rc = launch_dq<T, DP, 1, 1>(a, st);
    else if constexpr (sizeof(T) == 4) rc = launch_dq<T, DP, 4, 1>(a, st);
    else if (rows <= 96) rc = launch_dq_wide<T, DP, 2>(a, st);
    else if (rows <= 512) rc = launch_dq_wide<T, DP, 4>(a, st);
    else rc = launch_dq_wide<T, DP, 8>(a, st);
    if (rc) return rc;
    if (keys <= 16) return launch_dkv<T, DP, 1, 1>(a, st);
    if constexpr (sizeof(T) == 4) return launch_dkv<T, DP, 4, 1>(a, st);
    else {
        if (keys <= 96) return launch_dkv_wide<T, DP, 2>(a, st);
        if (keys <= 512) return launch_dkv_wide<T, DP, 4>(a, st);
        return launch_dkv_wide<T, DP, 8>(a, st);
    }
}

template <typename T>
int fwd(const AttnArgs& a, hipStream_t st) {
    if (a.dim <= 32) return fwd_dim<T, 32>(a, st);
    if (a.dim <= 64) return fwd_dim<T, 64>(a, st);
    return fwd_dim<T, 128>(a, st);
}

template <typename T>
int bwd(const AttnArgs& a, hipStream_t st) {
    const long long rows = (long long)a.tokens_q * a.heads;
    if (rows > 0) hipLaunchKernelGGL((delta_kernel<T>), dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, st, a);
    if (a.dim <= 32) return bwd_dim<T, 32>(a, st);
    if (a.dim <= 64) return bwd_dim<T, 64>(a, st);
    return bwd_dim<T, 128>(a, st);
}

}  // namespace attn
}  // namespace icap
