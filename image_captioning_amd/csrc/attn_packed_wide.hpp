// The 16-bit forms of the attention kernels for sequences of more than 16 rows (attn_packed.hpp: the mathematics, the fp32
// forms and the one-wave forms).  The same transposed products on 32 x 32 x 16 matrix instructions: a wave owns 32 rows (or, for
// dK and dV, 32 keys) in registers, a query (key) is column lane % 32 of every accumulator, and the eight values a lane half holds of
// 16 accumulator rows are the B operand of the next product as they come.
// What bounds them: a wave reads each staged tile whole, 1 KB a matrix instruction of 32 cycles, so that at four waves a CU the LDS
// (128 bytes a cycle) and the matrix cores are level, and the exponentials (16 cycles a wave each) take as long again at
// dim 128; the kernels therefore want two waves a SIMD that interleave, and nothing else in the loop:
//   * tiles go global -> LDS without registers, double-buffered, one barrier a step;
//   * LDS rows are not padded (the direct loads write linearly) but permuted in 16-byte slots by swizzle(), which spreads the 8
//     rows of a fragment read and the 4 rows of a transposing read over different banks;
//   * the running maximum is only followed when it grows by more than 2^8 (weights stay below 256, sums in fp32, so nothing
//     is lost), which leaves the accumulators alone in almost every step.
#pragma once
#include "attn_packed.hpp"

namespace icap {
namespace attn {

__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// permutation of a row's 16-byte slots: rows of 256, 128 and 64 bytes share a bank line of 256 bytes one, two and four at a time
template <int DP>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (DP == 128) return ((row & 3) << 1) | ((row >> 2) & 1);
    else if constexpr (DP == 64) return (((row >> 1) & 1) << 1) | ((row >> 2) & 1);
    else return (row >> 2) & 1;
}

// [ROWS][DP] of 16-bit values, global -> LDS
template <typename T, int ROWS, int DP, int NTHR>
struct Direct {
    static constexpr int CH = DP / 8, PIECES = ROWS * CH, N = PIECES < NTHR ? 1 : PIECES / NTHR;
    static_assert(PIECES < NTHR ? PIECES % 64 == 0 : PIECES % NTHR == 0, "whole passes, or whole waves of one");
    int row[N], col[N];
    __device__ __forceinline__ void init(int dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + i * NTHR;
            row[i] = c / CH;
            const int s = ((c % CH) ^ swizzle<DP>(row[i])) * 8;
            col[i] = s < dim ? s : 0;           // columns behind dim meet zeros of the other operand
        }
    }
    __device__ __forceinline__ void put(const T* p, int i, T* lds) const {
        if (PIECES < NTHR && threadIdx.x >= PIECES) return;         // a short tile does not need every wave
        __builtin_amdgcn_global_load_lds(p, (__attribute__((address_space(3))) void*)(lds + ((threadIdx.x >> 6) * 64 + i * NTHR) * 8), 16, 0, 0);
    }
    // rows `stride` apart; those behind `valid` (>= 1) repeat the last one (masked)
    __device__ __forceinline__ void load(const T* src, int stride, int valid, T* lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i) put(src + (unsigned)(min(row[i], valid - 1) * stride + col[i]), i, lds);
    }
    // rows that are (token, head of the group) pairs
    __device__ __forceinline__ void load_rows(const T* src, int tok, int head, int group, int row0, int nrow, T* lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = min(row0 + row[i], nrow - 1), t = r / group;
            put(src + (long long)t * tok + ((r - t * group) * head + col[i]), i, lds);
        }
    }
};

__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// row row0 + lane % 32, columns 16 kk + 8 (lane / 32) .. + 7
template <typename T, int DP>
__device__ __forceinline__ typename Vec<T>::x8 row_frag32(const T* lds, int row0, int kk) {
    const int lane = threadIdx.x & 63, r = lane & 31, lh = lane >> 5;
    return *reinterpret_cast<const typename Vec<T>::x8*>(lds + (row0 + r) * DP + (((kk * 2 + lh) ^ swizzle<DP>(r)) * 8));
}

// transposed: matrix row = tile column col0 + lane % 32; contraction over 16 tile rows in the order of an accumulator's eight
// registers: rows {0-3, 8-11} + 4 (lane / 32)
template <typename T, int DP>
__device__ __forceinline__ typename Vec<T>::x8 col_frag32(const T* lds, int row0, int col0) {
    const int lane = threadIdx.x & 63, l = lane & 15, half = (lane >> 4) & 1, lh = lane >> 5;
    const int r = 4 * lh + (l >> 2);
    const int slot = (col0 >> 3) + half * 2 + ((l & 3) >> 1);
    const T* p = lds + (row0 + r) * DP + (slot ^ swizzle<DP>(r)) * 8 + (l & 1) * 4;
    typedef __attribute__((address_space(3))) i16x4* lds_ptr;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 8 * DP));
    typedef short i16x8 __attribute__((ext_vector_type(8)));
    const i16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Vec<T>::x8, both);
}

// eight registers of an accumulator (16 of its rows) as an operand
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 acc_frag32(const f32x16& a, int half) {
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = a[half * 8 + e];
    return __builtin_convertvector(x, typename Vec<T>::x8);
}

template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 global_frag32(const T* row, int kk, int dim, bool ok) {
    const int col = kk * 16 + ((threadIdx.x & 63) >> 5) * 8;
    typename Vec<T>::x8 f = *reinterpret_cast<const typename Vec<T>::x8*>(row + (col < dim ? col : 0));
    if (!(ok && col < dim)) f = typename Vec<T>::x8{};
    return f;
}

// accumulator row of register e
__device__ __forceinline__ constexpr int acc_row(int e) { return (e & 3) + 8 * (e >> 2); }

__device__ __forceinline__ f32x16 zeros16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}

// one lane's 16 values of a result row (columns col0 + acc_row(e) + 4 (lane / 32)), four at a time
template <typename T>
__device__ __forceinline__ void store16(T* p, int col0, int dim, const f32x16& v, float f) {
    const int lh = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = col0 + 8 * g + 4 * lh;
        if (d < dim) store4<T>(p + d, f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]} * f);
    }
}

// this lane's row of a tile of (token, head) rows, and what it and its wave see
struct Row { int tok, hd, see, wkeys, wfull; bool ok; };
__device__ __forceinline__ Row row_of(const AttnArgs& a, int row0, int nrow, int nq, int nk) {
    const int r = row0 + (threadIdx.x & 31), rr = min(r, nrow - 1), off = nk - nq;
    Row w;
    w.ok = r < nrow;
    w.tok = rr / a.group;
    w.hd = rr - w.tok * a.group;
    w.see = w.ok ? (a.causal ? min(nk, max(w.tok + off + 1, 0)) : nk) : 0;
    const int last = min((row0 + 31) / a.group, nq - 1);
    w.wkeys = row0 < nrow ? (a.causal ? min(nk, max(last + off + 1, 0)) : nk) : 0;
    w.wfull = row0 + 32 <= nrow ? (a.causal ? min(nk, max(row0 / a.group + off + 1, 0)) : nk) : 0;
    return w;
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 2 && DP == 128 ? 1 : 2) void fwd_wide_kernel(const AttnArgs a) {
    constexpr int NTHR = NW * 64, BM = NW * 32, BN = 64, KK = DP / 16, ND = DP / 32;
    __shared__ __attribute__((aligned(1024))) T sk[2][BN * DP];
    __shared__ __attribute__((aligned(1024))) T sv[2][BN * DP];
    __shared__ int sh[16];
    const int kvh = blockIdx.x % a.kv_heads, bid = blockIdx.x / a.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lh = lane >> 5;
    const Where w = locate<NTHR>(a.cu_q, a.seqs, a.tokens_q, a.group, BM, bid, sh);
    if (w.seq < 0) {
        if (kvh == 0) {
            int b0, n0;
            range_of(a.cu_q, a.seqs - 1, a.tokens_q, b0, n0);
            clear_behind<T, NTHR>((T*)a.out, a.lse, b0 + n0, a.tokens_q, a.heads, a.dim, bid - w.used, gridDim.x / a.kv_heads - w.used);
        }
        return;
    }
    int q0, nq, k0, nk;
    range_of(a.cu_q, w.seq, a.tokens_q, q0, nq);
    range_of(a.cu_k, w.seq, a.tokens_k, k0, nk);
    const int nrow = nq * a.group, tiles = (nrow + BM - 1) / BM, tile = a.causal ? tiles - 1 - w.tile : w.tile;
    const int row0 = tile * BM + wave * 32;
    const Row me = row_of(a, row0, nrow, nq, nk);
    const T* qp = (const T*)a.q + (long long)(q0 + me.tok) * a.q_tok + (long long)(kvh * a.group + me.hd) * a.q_head;
    const T* kb = (const T*)a.k + (long long)k0 * a.k_tok + (long long)kvh * a.k_head;
    const T* vb = (const T*)a.v + (long long)k0 * a.v_tok + (long long)kvh * a.v_head;
    typename Vec<T>::x8 qf[KK];
#pragma unroll
    for (int c = 0; c < KK; ++c) qf[c] = global_frag32<T>(qp, c, a.dim, me.ok);
    const int last = min((tile * BM + BM - 1) / a.group, nq - 1);
    const int keys = a.causal ? min(nk, max(last + nk - nq + 1, 0)) : nk;

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = zeros16();
    float m = -INFINITY, l = 0.f;
    const float c2 = a.scale * LOG2E;
    Direct<T, BN, DP, NTHR> dir;
    dir.init(a.dim);
    if (keys > 0) {
        dir.load(kb, (int)a.k_tok, nk, sk[0]);
        dir.load(vb, (int)a.v_tok, nk, sv[0]);
    }
    int buf = 0;
    for (int n0 = 0; n0 < keys; n0 += BN, buf ^= 1) {
        landed();
        if (n0 + BN < keys) {
            dir.load(kb + (long long)(n0 + BN) * a.k_tok, (int)a.k_tok, nk - n0 - BN, sk[buf ^ 1]);
            dir.load(vb + (long long)(n0 + BN) * a.v_tok, (int)a.v_tok, nk - n0 - BN, sv[buf ^ 1]);
        }
        if (n0 >= me.wkeys) continue;
        f32x16 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            s[kt] = zeros16();
#pragma unroll
            for (int c = 0; c < KK; ++c) s[kt] = mma32(row_frag32<T, DP>(sk[buf], kt * 32, c), qf[c], s[kt]);
        }
        if (n0 + BN > me.wfull) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (n0 + kt * 32 + acc_row(e) + 4 * lh >= me.see) s[kt][e] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kt][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 32)) * c2;
        if (__any(mx > m + 8.0f)) {
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kt][e] = __builtin_amdgcn_exp2f(fmaf(s[kt][e], c2, -base));
                sum += s[kt][e];
            }
        l += sum;
        // P is rounded to T for the matrix cores (2^-9 / 2^-12 of each weight, as much as the result's own rounding); l is not
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const auto pf = acc_frag32<T>(s[j >> 1], j & 1);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = mma32(col_frag32<T, DP>(sv[buf], j * 16, d * 32), pf, o[d]);
        }
    }
    const float sum = l + __shfl_xor(l, 32);
    if (!me.ok) return;
    const long long at = (long long)(q0 + me.tok) * a.heads + kvh * a.group + me.hd;
    const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
    for (int d = 0; d < ND; ++d) store16<T>((T*)a.out + at * a.dim, d * 32, a.dim, o[d], inv);
    if (lh == 0 && a.lse) a.lse[at] = sum > 0.f ? fmaf(m, LN2, logf(sum)) : (sum == 0.f ? -INFINITY : sum);
}

// ------------------------------------------------------------------------------------------------ dQ
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 2 && DP == 128 ? 1 : 2) void dq_wide_kernel(const AttnArgs a) {
    constexpr int NTHR = NW * 64, BM = NW * 32, BN = 64, KK = DP / 16, ND = DP / 32;
    __shared__ __attribute__((aligned(1024))) T sk[2][BN * DP];
    __shared__ __attribute__((aligned(1024))) T sv[2][BN * DP];
    __shared__ int sh[16];
    const int kvh = blockIdx.x % a.kv_heads, bid = blockIdx.x / a.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lh = lane >> 5;
    const Where w = locate<NTHR>(a.cu_q, a.seqs, a.tokens_q, a.group, BM, bid, sh);
    if (w.seq < 0) {
        if (kvh == 0) {
            int b0, n0;
            range_of(a.cu_q, a.seqs - 1, a.tokens_q, b0, n0);
            clear_behind<T, NTHR>((T*)a.dq, nullptr, b0 + n0, a.tokens_q, a.heads, a.dim, bid - w.used, gridDim.x / a.kv_heads - w.used);
        }
        return;
    }
    int q0, nq, k0, nk;
    range_of(a.cu_q, w.seq, a.tokens_q, q0, nq);
    range_of(a.cu_k, w.seq, a.tokens_k, k0, nk);
    const int nrow = nq * a.group, tiles = (nrow + BM - 1) / BM, tile = a.causal ? tiles - 1 - w.tile : w.tile;
    const int row0 = tile * BM + wave * 32;
    const Row me = row_of(a, row0, nrow, nq, nk);
    const int head = kvh * a.group + me.hd;
    const long long at = (long long)(q0 + me.tok) * a.heads + head;
    const T* qp = (const T*)a.q + (long long)(q0 + me.tok) * a.q_tok + (long long)head * a.q_head;
    const T* gp = (const T*)a.dout + (long long)(q0 + me.tok) * a.g_tok + (long long)head * a.g_head;
    const T* kb = (const T*)a.k + (long long)k0 * a.k_tok + (long long)kvh * a.k_head;
    const T* vb = (const T*)a.v + (long long)k0 * a.v_tok + (long long)kvh * a.v_head;
    const float lse2 = a.lse[at] * LOG2E, delta = a.delta[at], c2 = a.scale * LOG2E;
    typename Vec<T>::x8 qf[KK], gf[KK];
#pragma unroll
    for (int c = 0; c < KK; ++c) {
        qf[c] = global_frag32<T>(qp, c, a.dim, me.ok);
        gf[c] = global_frag32<T>(gp, c, a.dim, me.ok);
    }
    const int last = min((tile * BM + BM - 1) / a.group, nq - 1);
    const int keys = a.causal ? min(nk, max(last + nk - nq + 1, 0)) : nk;
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[d] = zeros16();
    Direct<T, BN, DP, NTHR> dir;
    dir.init(a.dim);
    if (keys > 0) {
        dir.load(kb, (int)a.k_tok, nk, sk[0]);
        dir.load(vb, (int)a.v_tok, nk, sv[0]);
    }
    int buf = 0;
    for (int n0 = 0; n0 < keys; n0 += BN, buf ^= 1) {
        landed();
        if (n0 + BN < keys) {
            dir.load(kb + (long long)(n0 + BN) * a.k_tok, (int)a.k_tok, nk - n0 - BN, sk[buf ^ 1]);
            dir.load(vb + (long long)(n0 + BN) * a.v_tok, (int)a.v_tok, nk - n0 - BN, sv[buf ^ 1]);
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            if (n0 + kt * 32 >= me.wkeys) break;
            f32x16 s = zeros16(), dp = zeros16();
#pragma unroll
            for (int c = 0; c < KK; ++c) {
                s = mma32(row_frag32<T, DP>(sk[buf], kt * 32, c), qf[c], s);
                dp = mma32(row_frag32<T, DP>(sv[buf], kt * 32, c), gf[c], dp);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, -lse2)) * (dp[e] - delta);
            if (n0 + kt * 32 + 32 > me.wfull) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (n0 + kt * 32 + acc_row(e) + 4 * lh >= me.see) s[e] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const auto df = acc_frag32<T>(s, j);            // one rounding of dS to T, as of P
#pragma unroll
                for (int d = 0; d < ND; ++d) dq[d] = mma32(col_frag32<T, DP>(sk[buf], kt * 32 + j * 16, d * 32), df, dq[d]);
            }
        }
    }
    if (!me.ok) return;
#pragma unroll
    for (int d = 0; d < ND; ++d) store16<T>((T*)a.dq + at * a.dim, d * 32, a.dim, dq[d], a.scale);
}

// ------------------------------------------------------------------------------------------------ dK, dV
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, 2) void dkv_wide_kernel(const AttnArgs a) {
    constexpr int NTHR = NW * 64, BK = NW * 32, BR = 32, KK = DP / 16, ND = DP / 32;
    __shared__ __attribute__((aligned(1024))) T sq[2][BR * DP];
    __shared__ __attribute__((aligned(1024))) T sg[2][BR * DP];
    __shared__ __attribute__((aligned(16))) float srow[2][3][BR];       // lse, delta, number of keys seen
    __shared__ int sh[16];
    const int kvh = blockIdx.x % a.kv_heads, bid = blockIdx.x / a.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lh = lane >> 5;
    const Where w = locate<NTHR>(a.cu_k, a.seqs, a.tokens_k, 1, BK, bid, sh);
    if (w.seq < 0) {
        if (kvh == 0) {
            int b0, n0;
            range_of(a.cu_k, a.seqs - 1, a.tokens_k, b0, n0);
            clear_behind<T, NTHR>((T*)a.dk, nullptr, b0 + n0, a.tokens_k, a.kv_heads, a.dim, bid - w.used, gridDim.x / a.kv_heads - w.used);
            clear_behind<T, NTHR>((T*)a.dv, nullptr, b0 + n0, a.tokens_k, a.kv_heads, a.dim, bid - w.used, gridDim.x / a.kv_heads - w.used);
        }
        return;
    }
    int q0, nq, k0, nk;
    range_of(a.cu_q, w.seq, a.tokens_q, q0, nq);
    range_of(a.cu_k, w.seq, a.tokens_k, k0, nk);
    const int nrow = nq * a.group, off = nk - nq, key0 = w.tile * BK + wave * 32, key = key0 + (lane & 31);
    const T* qb = (const T*)a.q + (long long)q0 * a.q_tok + (long long)kvh * a.group * a.q_head;
    const T* gb = (const T*)a.dout + (long long)q0 * a.g_tok + (long long)kvh * a.group * a.g_head;
    typename Vec<T>::x8 kf[KK], vf[KK];
    {
        const long long kk = k0 + min(key, nk - 1);
        const T* kp = (const T*)a.k + kk * a.k_tok + (long long)kvh * a.k_head;
        const T* vp = (const T*)a.v + kk * a.v_tok + (long long)kvh * a.v_head;
#pragma unroll
        for (int c = 0; c < KK; ++c) {
            kf[c] = global_frag32<T>(kp, c, a.dim, key < nk);
            vf[c] = global_frag32<T>(vp, c, a.dim, key < nk);
        }
    }
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zeros16();
    const float c2 = a.scale * LOG2E;
    // the first row that sees the workgroup's first key
    const int first = a.causal ? min(max(w.tile * BK - off, 0), nq) * a.group / BR * BR : 0;
    Direct<T, BR, DP, NTHR> dir;
    dir.init(a.dim);
    auto fetch = [&](int r0, int buf) __attribute__((always_inline)) {
        dir.load_rows(qb, (int)a.q_tok, (int)a.q_head, a.group, r0, nrow, sq[buf]);
        dir.load_rows(gb, (int)a.g_tok, (int)a.g_head, a.group, r0, nrow, sg[buf]);
        if (threadIdx.x < BR) {
            const int r = r0 + threadIdx.x, rr = min(r, nrow - 1), t = rr / a.group;
            const long long at = (long long)(q0 + t) * a.heads + kvh * a.group + (rr - t * a.group);
            srow[buf][0][threadIdx.x] = a.lse[at] * LOG2E;
            srow[buf][1][threadIdx.x] = a.delta[at];
            srow[buf][2][threadIdx.x] = __int_as_float(r < nrow ? (a.causal ? min(nk, max(t + off + 1, 0)) : nk) : 0);
        }
    };
    if (first < nrow) fetch(first, 0);
    int buf = 0;
    for (int r0 = first; r0 < nrow; r0 += BR, buf ^= 1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        landed();
        if (r0 + BR < nrow) fetch(r0 + BR, buf ^ 1);
        // whole when every row of the step sees every key of the wave, nothing to do when none sees any
        const int see0 = a.causal ? min(nk, max(r0 / a.group + off + 1, 0)) : nk;
        const int see1 = a.causal ? min(nk, max(min(r0 + BR - 1, nrow - 1) / a.group + off + 1, 0)) : nk;
        if (key0 >= see1) continue;
        f32x16 s = zeros16(), dp = zeros16();
#pragma unroll
        for (int c = 0; c < KK; ++c) {
            s = mma32(row_frag32<T, DP>(sq[buf], 0, c), kf[c], s);
            dp = mma32(row_frag32<T, DP>(sg[buf], 0, c), vf[c], dp);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(&srow[buf][0][8 * g + 4 * lh]), d4 = *reinterpret_cast<const f32x4*>(&srow[buf][1][8 * g + 4 * lh]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = 4 * g + i;
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, -l4[i]));
                dp[e] = s[e] * (dp[e] - d4[i]);
            }
        }
        if (key0 + 32 > see0 || r0 + BR > nrow) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (key >= __float_as_int(srow[buf][2][acc_row(e) + 4 * lh])) s[e] = dp[e] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const auto pf = acc_frag32<T>(s, j), df = acc_frag32<T>(dp, j);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                dv[d] = mma32(col_frag32<T, DP>(sg[buf], j * 16, d * 32), pf, dv[d]);
                dk[d] = mma32(col_frag32<T, DP>(sq[buf], j * 16, d * 32), df, dk[d]);
            }
        }
    }
    if (key >= nk) return;
    const long long at = ((long long)(k0 + key) * a.kv_heads + kvh) * a.dim;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        store16<T>((T*)a.dk + at, d * 32, a.dim, dk[d], a.scale);
        store16<T>((T*)a.dv + at, d * 32, a.dim, dv[d], 1.0f);
    }
}

template <typename T, int DP, int NW>
int launch_fwd_wide(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((fwd_wide_kernel<T, DP, NW>), dim3(blocks_for(a, (long long)a.tokens_q * a.group, NW * 32)), dim3(NW * 64), 0, st, a);
    return launch_status("attention_packed_fwd");
}
template <typename T, int DP, int NW>
int launch_dq_wide(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((dq_wide_kernel<T, DP, NW>), dim3(blocks_for(a, (long long)a.tokens_q * a.group, NW * 32)), dim3(NW * 64), 0, st, a);
    return launch_status("attention_packed_bwd");
}
template <typename T, int DP, int NW>
int launch_dkv_wide(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((dkv_wide_kernel<T, DP, NW>), dim3(blocks_for(a, a.tokens_k, NW * 32)), dim3(NW * 64), 0, st, a);
    return launch_status("attention_packed_bwd");
}

}  // namespace attn
}  // namespace icap
