// Attention over packed sequences (no padding: sequence b owns rows cu[b] .. cu[b + 1] of the packed tensors), forward and
// gradients, for one element type T.
//   S = scale q k^T (keys after a query's place hidden when causal, places aligned at the sequences' ENDS), P = softmax(S), O = P V
//   dV = P^T dO,  dS = P (dO V^T - rowsum(dO O)),  dQ = scale dS K,  dK = scale dS^T Q
// Query heads that share a key head are rows of one matrix: row r of a sequence is (token r / group, head r % group).  A key
// is then read once for the whole group, the single-token form fills a 16-row tile with its group, and dK / dV sum over the
// group inside one workgroup, in a fixed order, without atomics.
// One pass over the keys with a running maximum and sum.  The products are formed transposed (S^T = K Q^T, O^T = V^T P^T), so
// that a query is a column (lane % 16) of every accumulator: its maximum, sum and rescaling stay in the lane, and the
// accumulator of S^T is, register for register, the B operand of the next product (its 4-row groups only permute the
// contraction, and V^T is read in the same order).  Rows that see no key get zeros (and a log-sum of -inf).
#pragma once
#include "packed.hpp"

namespace icap {
namespace attn {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

template <typename T> struct Tile {
    static constexpr int PAD = 16 / sizeof(T);      // one 16-byte slot a row: the 16 rows of a fragment read start in different banks
};

// rows of 16-byte pieces: [ROWS][DP] of a packed tensor between global memory and LDS, through registers
template <typename T, int ROWS, int DP, int NTHR>
struct Stage {
    static constexpr int EPC = 16 / sizeof(T), CH = DP / EPC, N = (ROWS * CH + NTHR - 1) / NTHR, LD = DP + Tile<T>::PAD;
    u32x4 r[N];
    // src: row 0, rows `stride` elements apart; valid >= 1 rows exist, the others and columns from dim on become zeros
    __device__ __forceinline__ void load(const T* src, long long stride, int valid, int dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + i * NTHR, row = c / CH, col = (c % CH) * EPC;
            const T* p = src + (long long)min(row, valid - 1) * stride + (col < dim ? col : 0);
            u32x4 x = *reinterpret_cast<const u32x4*>(p);
            const unsigned keep = (row < valid && col < dim) ? 0xffffffffu : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] &= keep;
            r[i] = x;
        }
    }
    // rows that are (token, head of the group) pairs
    __device__ __forceinline__ void load_rows(const T* src, long long tok, long long head, int group, int row0, int nrow, int dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + i * NTHR, row = row0 + c / CH, col = (c % CH) * EPC;
            const int rr = min(row, nrow - 1), t = rr / group;
            const T* p = src + (long long)t * tok + (long long)(rr - t * group) * head + (col < dim ? col : 0);
            u32x4 x = *reinterpret_cast<const u32x4*>(p);
            const unsigned keep = (row < nrow && col < dim) ? 0xffffffffu : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] &= keep;
            r[i] = x;
        }
    }
    __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + i * NTHR;
            if (ROWS * CH % NTHR != 0 && c >= ROWS * CH) break;
            *reinterpret_cast<u32x4*>(lds + (c / CH) * LD + (c % CH) * EPC) = r[i];
        }
    }
};

// fragment of a row-major LDS tile whose rows are the matrix rows: row row0 + lane % 16, columns 32 c + 8 (lane / 16) .. + 7
template <typename T, int LD>
__device__ __forceinline__ typename Vec<T>::x8 row_frag(const T* lds, int row0, int c) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const typename Vec<T>::x8*>(lds + (row0 + (lane & 15)) * LD + c * 32 + (lane >> 4) * 8);
}

// fragment of the same tile transposed: matrix row = tile column col0 + lane % 16; the contraction runs over the 32 tile rows
// from row0, in the order of an accumulator's registers: slots 0-3 are rows 4 (lane / 16) + 0..3, slots 4-7 the same + 16.
// 16-bit types: the transposing LDS read, which hands lane l of 16 column l of the 4 x 16 block its 16 lanes address.
template <typename T, int LD>
__device__ __forceinline__ typename Vec<T>::x8 col_frag(const T* lds, int row0, int col0) {
    const int lane = threadIdx.x & 63, l = lane & 15, grp = lane >> 4;
    if constexpr (sizeof(T) == 2) {
        const T* p = lds + (row0 + grp * 4 + (l >> 2)) * LD + col0 + (l & 3) * 4;
        typedef __attribute__((address_space(3))) i16x4* lds_ptr;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 16 * LD));
        typedef short i16x8 __attribute__((ext_vector_type(8)));
        const i16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(typename Vec<T>::x8, both);
    } else {
        const T* p = lds + (row0 + grp * 4) * LD + col0 + l;
        typename Vec<T>::x8 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[j] = p[j * LD]; f[4 + j] = p[(16 + j) * LD]; }
        return f;
    }
}

// two accumulators (tile rows 0-15 and 16-31 of a 32-row step) as the operand of the product that contracts those rows
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 acc_frag(f32x4 a, f32x4 b) {
    if constexpr (sizeof(T) == 4) return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    else return __builtin_convertvector(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), typename Vec<T>::x8);
}

// fragment of a global row: columns 32 c + 8 (lane / 16) .. + 7, zeros from dim on and when !ok (p stays readable)
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 global_frag(const T* row, int c, int dim, bool ok) {
    const int col = c * 32 + ((threadIdx.x & 63) >> 4) * 8;
    typename Vec<T>::x8 f = *reinterpret_cast<const typename Vec<T>::x8*>(row + (col < dim ? col : 0));
    if (!(ok && col < dim)) f = typename Vec<T>::x8{};
    return f;
}

struct Where { int seq, tile, used; };

// Which sequence and which of its tiles workgroup `bid` owns, from the running sum of the sequences' tile counts; every thread
// looks at one sequence.  seq = -1: behind the last tile; used = the number of tiles there are.  Lengths are bounded by
// `tokens`, so a wrong list of offsets reads and writes nothing outside the tensors.  sh: 16 ints of LDS.
template <int NTHR>
__device__ __forceinline__ Where locate(const int* cu, int seqs, int tokens, int per_token, int rows, int bid, int* sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int base = 0;
    for (int s0 = 0; s0 < seqs; s0 += NTHR) {
        const int s = s0 + tid;
        int n = 0;
        if (s < seqs) {
            const int a = min(max(cu[s], 0), tokens), b = min(max(cu[s + 1], a), tokens);
            n = ((b - a) * per_token + rows - 1) / rows;
        }
        int inc = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int t = __shfl_up(inc, d); if (lane >= d) inc += t; }
        if (lane == 63) sh[wave] = inc;
        if (tid == 0) sh[8] = -1;
        __syncthreads();
        int pre = 0, tot = 0;
#pragma unroll
        for (int w = 0; w < NTHR / 64; ++w) { const int t = sh[w]; if (w < wave) pre += t; tot += t; }
        const int end = base + pre + inc;
        if (n > 0 && bid < end && bid >= end - n) { sh[8] = s; sh[9] = bid - (end - n); }
        __syncthreads();
        const int found = sh[8], tile = sh[9];
        __syncthreads();
        if (found >= 0) return {__builtin_amdgcn_readfirstlane(found), __builtin_amdgcn_readfirstlane(tile), 0};
        base += tot;
    }
    return {-1, 0, base};
}

__device__ __forceinline__ void range_of(const int* cu, int s, int tokens, int& begin, int& n) {
    begin = min(max(cu[s], 0), tokens);
    n = min(max(cu[s + 1], begin), tokens) - begin;
}

// rows that belong to no sequence (behind the last one) get zeros, from the workgroups that own no tile
template <typename T, int NTHR>
__device__ __forceinline__ void clear_behind(T* dst, float* lse, int first, int tokens, int heads, int dim, int id, int ids) {
    const long long per = (long long)heads * dim, n = (tokens - first) * per;
    T* p = dst + first * per;
    for (long long i = (long long)id * NTHR + threadIdx.x; i < n / 8; i += (long long)ids * NTHR)
        *reinterpret_cast<typename Vec<T>::x8*>(p + i * 8) = typename Vec<T>::x8{};
    if (lse)
        for (long long i = (long long)id * NTHR + threadIdx.x; i < (long long)(tokens - first) * heads; i += (long long)ids * NTHR)
            lse[(long long)first * heads + i] = -INFINITY;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
    else *reinterpret_cast<typename Vec<T>::x4*>(p) = __builtin_convertvector(v, typename Vec<T>::x4);
}

__device__ __forceinline__ float across_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float across_groups_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Split keys: workgroup z takes a share of the keys (whole steps, at least two of them, so that short sequences are not split)
template <int BN>
__device__ __forceinline__ void split_range(int keys, int splits, int z, int& lo, int& hi) {
    const int steps = (keys + BN - 1) / BN, per = max((steps + splits - 1) / splits, splits > 1 ? 2 : 1) * BN;
    lo = min(z * per, keys);
    hi = min(lo + per, keys);
}

// ------------------------------------------------------------------------------------------------ forward
// NW waves of NT x 16 rows each; 64 keys a step, staged through registers while the step before multiplies
template <typename T, int DP, int NW, int NT>
__global__ __launch_bounds__(NW * 64) void fwd_kernel(const AttnArgs a) {
    constexpr int NTHR = NW * 64, BM = NW * NT * 16, BN = 64, LD = DP + Tile<T>::PAD, CK = DP / 32, CD = DP / 16;
    __shared__ __attribute__((aligned(16))) T sk[BN * LD];
    __shared__ __attribute__((aligned(16))) T sv[BN * LD];
    __shared__ int sh[16];
    const int kvh = blockIdx.x % a.kv_heads, bid = blockIdx.x / a.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 4;
    const Where w = locate<NTHR>(a.cu_q, a.seqs, a.tokens_q, a.group, BM, bid, sh);
    if (w.seq < 0) {
        if (kvh == 0 && blockIdx.y == 0) {
            int b0, n0;
            range_of(a.cu_q, a.seqs - 1, a.tokens_q, b0, n0);
            clear_behind<T, NTHR>((T*)a.out, a.lse, b0 + n0, a.tokens_q, a.heads, a.dim, bid - w.used, gridDim.x / a.kv_heads - w.used);
        }
        return;
    }
    int q0, nq, k0, nk;
    range_of(a.cu_q, w.seq, a.tokens_q, q0, nq);
    range_of(a.cu_k, w.seq, a.tokens_k, k0, nk);
    const int nrow = nq * a.group, tiles = (nrow + BM - 1) / BM;
    const int tile = a.causal ? tiles - 1 - w.tile : w.tile;            // the longest tiles of a sequence start first
    const int row0 = tile * BM + wave * NT * 16, off = nk - nq;
    const T* qb = (const T*)a.q + (long long)q0 * a.q_tok + (long long)kvh * a.group * a.q_head;
    const T* kb = (const T*)a.k + (long long)k0 * a.k_tok + (long long)kvh * a.k_head;
    const T* vb = (const T*)a.v + (long long)k0 * a.v_tok + (long long)kvh * a.v_head;

    int tok[NT], hd[NT], see[NT];           // this lane's row: token, head of the group, number of keys it sees
    typename Vec<T>::x8 qf[NT][CK];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + t * 16 + (lane & 15), rr = min(r, nrow - 1);
        tok[t] = rr / a.group;
        hd[t] = rr - tok[t] * a.group;
        see[t] = r < nrow ? (a.causal ? min(nk, max(tok[t] + off + 1, 0)) : nk) : 0;
        const T* p = qb + (long long)tok[t] * a.q_tok + (long long)hd[t] * a.q_head;
#pragma unroll
        for (int c = 0; c < CK; ++c) qf[t][c] = global_frag<T>(p, c, a.dim, r < nrow);
    }
    // keys that any row of the workgroup sees, any row of this wave sees, and all rows of this wave see (no mask needed there)
    const int last = min((tile * BM + BM - 1) / a.group, nq - 1);
    const int keys = a.causal ? min(nk, max(last + off + 1, 0)) : nk;
    const int wlast = min((row0 + NT * 16 - 1) / a.group, nq - 1);
    const int wkeys = row0 < nrow ? (a.causal ? min(nk, max(wlast + off + 1, 0)) : nk) : 0;
    const int wfull = row0 + NT * 16 <= nrow ? (a.causal ? min(nk, max(row0 / a.group + off + 1, 0)) : nk) : 0;
    int lo, hi;
    split_range<BN>(keys, a.splits, blockIdx.y, lo, hi);

    f32x4 o[CD][NT];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < CD; ++d) o[d][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float c2 = a.scale * LOG2E;
    Stage<T, BN, DP, NTHR> stk, stv;
    if (lo < hi) {
        stk.load(kb + (long long)lo * a.k_tok, a.k_tok, nk - lo, a.dim);
        stv.load(vb + (long long)lo * a.v_tok, a.v_tok, nk - lo, a.dim);
    }
    for (int n0 = lo; n0 < hi; n0 += BN) {
        stk.store(sk);
        stv.store(sv);
        __syncthreads();
        if (n0 + BN < hi) {
            stk.load(kb + (long long)(n0 + BN) * a.k_tok, a.k_tok, nk - n0 - BN, a.dim);
            stv.load(vb + (long long)(n0 + BN) * a.v_tok, a.v_tok, nk - n0 - BN, a.dim);
        }
        if (n0 < wkeys) {
            f32x4 s[4][NT];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
                for (int t = 0; t < NT; ++t) s[kt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CK; ++c) {
                    const auto kf = row_frag<T, LD>(sk, kt * 16, c);
#pragma unroll
                    for (int t = 0; t < NT; ++t) s[kt][t] = mma16(kf, qf[t][c], s[kt][t]);
                }
            }
            if (n0 + BN > wfull) {
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n0 + kt * 16 + grp * 4 + i >= see[t]) s[kt][t][i] = -INFINITY;
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float mx = s[0][t][0];
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[kt][t][i]);
                mx = across_groups_max(mx);
                const float mn = fmaxf(m[t], mx * c2);
                const float base = mn == -INFINITY ? 0.f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[t] - base);
                m[t] = mn;
                float sum = 0.f;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(s[kt][t][i], c2, -base));
                        s[kt][t][i] = p;
                        sum += p;
                    }
                l[t] = fmaf(l[t], alpha, sum);
#pragma unroll
                for (int d = 0; d < CD; ++d) o[d][t] *= alpha;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // P is rounded to T for the matrix cores (relative 2^-9 / 2^-12 of each weight, as much as the result's own rounding);
                // the sum l is taken from the unrounded values
                typename Vec<T>::x8 pf[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) pf[t] = acc_frag<T>(s[2 * h][t], s[2 * h + 1][t]);
#pragma unroll
                for (int d = 0; d < CD; ++d) {
                    const auto vf = col_frag<T, LD>(sv, h * 32, d * 16);
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[d][t] = mma16(vf, pf[t], o[d][t]);
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + t * 16 + (lane & 15);
        const float sum = across_groups_sum(l[t]);
        const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
        if (r >= nrow) continue;
        const long long at = (long long)(q0 + tok[t]) * a.heads + kvh * a.group + hd[t];
        const float lse = sum > 0.f ? fmaf(m[t], LN2, logf(sum)) : (sum == 0.f ? -INFINITY : sum);
        if (a.splits > 1) {
            const long long rows = (long long)a.tokens_q * a.heads;
            float* po = a.part + (rows * blockIdx.y + at) * a.dim;
#pragma unroll
            for (int d = 0; d < CD; ++d)
                if (d * 16 + grp * 4 < a.dim) *reinterpret_cast<f32x4*>(po + d * 16 + grp * 4) = o[d][t] * inv;
            if (grp == 0) a.part[rows * a.splits * a.dim + rows * blockIdx.y + at] = lse;
        } else {
            T* po = (T*)a.out + at * a.dim;
#pragma unroll
            for (int d = 0; d < CD; ++d)
                if (d * 16 + grp * 4 < a.dim) store4<T>(po + d * 16 + grp * 4, o[d][t] * inv);
            if (grp == 0 && a.lse) a.lse[at] = lse;
        }
    }
}

// joins the shares of split keys: each is a normalised result with its log-sum.  One group of DT threads per row.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const AttnArgs a) {
    const int per = a.dim / 4, rpb = 256 / per, i = threadIdx.x / per, d = (threadIdx.x - i * per) * 4;
    const long long rows = (long long)a.tokens_q * a.heads, used = (long long)min(max(a.cu_q[a.seqs], 0), a.tokens_q) * a.heads;
    const long long r = (long long)blockIdx.x * rpb + i;
    if (i >= rpb || r >= used) return;       // rows behind the last sequence were cleared by the first launch
    const float* pl = a.part + rows * a.splits * a.dim;
    float most = -INFINITY;
    for (int z = 0; z < a.splits; ++z) most = fmaxf(most, pl[rows * z + r]);
    const float base = most == -INFINITY ? 0.f : most;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    for (int z = 0; z < a.splits; ++z) {
        const float w = __builtin_amdgcn_exp2f((pl[rows * z + r] - base) * LOG2E);
        sum += w;
        acc += w * *reinterpret_cast<const f32x4*>(a.part + (rows * z + r) * a.dim + d);
    }
    const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
    store4<T>((T*)a.out + r * a.dim + d, acc * inv);
    if (d == 0 && a.lse) a.lse[r] = sum > 0.f ? base + logf(sum) : (sum == 0.f ? -INFINITY : sum);
}

// ------------------------------------------------------------------------------------------------ backward
// delta[row] = sum_d dO O, 8 lanes a row
template <typename T>
__global__ __launch_bounds__(256) void delta_kernel(const AttnArgs a) {
    const long long r = (long long)blockIdx.x * 32 + (threadIdx.x >> 3), rows = (long long)a.tokens_q * a.heads;
    const int part = threadIdx.x & 7;
    float s = 0.f;
    if (r < rows) {
        const long long t = r / a.heads;
        const T* g = (const T*)a.dout + t * a.g_tok + (r - t * a.heads) * a.g_head;
        const T* o = (const T*)a.o + r * a.dim;
        for (int d = part * 8; d < a.dim; d += 64) {
            const auto x = *reinterpret_cast<const typename Vec<T>::x8*>(g + d), y = *reinterpret_cast<const typename Vec<T>::x8*>(o + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf((float)x[e], (float)y[e], s);
        }
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    s += __shfl_xor(s, 4);
    if (part == 0 && r < rows) a.delta[r] = s;
}

// dQ: the forward's shape (rows in registers, keys staged), with dO beside Q and dS in P's place
template <typename T, int DP, int NW, int NT>
__global__ __launch_bounds__(NW * 64) void dq_kernel(const AttnArgs a) {
    constexpr int NTHR = NW * 64, BM = NW * NT * 16, BN = 32, LD = DP + Tile<T>::PAD, CK = DP / 32, CD = DP / 16;
    __shared__ __attribute__((aligned(16))) T sk[BN * LD];
    __shared__ __attribute__((aligned(16))) T sv[BN * LD];
    __shared__ int sh[16];
    const int kvh = blockIdx.x % a.kv_heads, bid = blockIdx.x / a.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 4;
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
    const int nrow = nq * a.group, tiles = (nrow + BM - 1) / BM;
    const int tile = a.causal ? tiles - 1 - w.tile : w.tile;
    const int row0 = tile * BM + wave * NT * 16, off = nk - nq;
    const T* qb = (const T*)a.q + (long long)q0 * a.q_tok + (long long)kvh * a.group * a.q_head;
    const T* gb = (const T*)a.dout + (long long)q0 * a.g_tok + (long long)kvh * a.group * a.g_head;
    const T* kb = (const T*)a.k + (long long)k0 * a.k_tok + (long long)kvh * a.k_head;
    const T* vb = (const T*)a.v + (long long)k0 * a.v_tok + (long long)kvh * a.v_head;
    int tok[NT], hd[NT], see[NT];
    float lse2[NT], delta[NT];
    typename Vec<T>::x8 qf[NT][CK], gf[NT][CK];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + t * 16 + (lane & 15), rr = min(r, nrow - 1);
        tok[t] = rr / a.group;
        hd[t] = rr - tok[t] * a.group;
        see[t] = r < nrow ? (a.causal ? min(nk, max(tok[t] + off + 1, 0)) : nk) : 0;
        const long long at = (long long)(q0 + tok[t]) * a.heads + kvh * a.group + hd[t];
        lse2[t] = a.lse[at] * LOG2E;
        delta[t] = a.delta[at];
        const T* p = qb + (long long)tok[t] * a.q_tok + (long long)hd[t] * a.q_head;
        const T* g = gb + (long long)tok[t] * a.g_tok + (long long)hd[t] * a.g_head;
#pragma unroll
        for (int c = 0; c < CK; ++c) {
            qf[t][c] = global_frag<T>(p, c, a.dim, r < nrow);
            gf[t][c] = global_frag<T>(g, c, a.dim, r < nrow);
        }
    }
    const int last = min((tile * BM + BM - 1) / a.group, nq - 1);
    const int keys = a.causal ? min(nk, max(last + off + 1, 0)) : nk;
    const int wlast = min((row0 + NT * 16 - 1) / a.group, nq - 1);
    const int wkeys = row0 < nrow ? (a.causal ? min(nk, max(wlast + off + 1, 0)) : nk) : 0;
    const int wfull = row0 + NT * 16 <= nrow ? (a.causal ? min(nk, max(row0 / a.group + off + 1, 0)) : nk) : 0;
    f32x4 dq[CD][NT];
#pragma unroll
    for (int d = 0; d < CD; ++d)
#pragma unroll
        for (int t = 0; t < NT; ++t) dq[d][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float c2 = a.scale * LOG2E;
    Stage<T, BN, DP, NTHR> stk, stv;
    if (keys > 0) {
        stk.load(kb, a.k_tok, nk, a.dim);
        stv.load(vb, a.v_tok, nk, a.dim);
    }
    for (int n0 = 0; n0 < keys; n0 += BN) {
        stk.store(sk);
        stv.store(sv);
        __syncthreads();
        if (n0 + BN < keys) {
            stk.load(kb + (long long)(n0 + BN) * a.k_tok, a.k_tok, nk - n0 - BN, a.dim);
            stv.load(vb + (long long)(n0 + BN) * a.v_tok, a.v_tok, nk - n0 - BN, a.dim);
        }
        if (n0 < wkeys) {
            f32x4 s[2][NT], dp[2][NT];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                for (int t = 0; t < NT; ++t) s[kt][t] = dp[kt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CK; ++c) {
                    const auto kf = row_frag<T, LD>(sk, kt * 16, c);
                    const auto vf = row_frag<T, LD>(sv, kt * 16, c);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        s[kt][t] = mma16(kf, qf[t][c], s[kt][t]);
                        dp[kt][t] = mma16(vf, gf[t][c], dp[kt][t]);
                    }
                }
            }
            const bool mask = n0 + BN > wfull;
            typename Vec<T>::x8 df[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float p = __builtin_amdgcn_exp2f(fmaf(s[kt][t][i], c2, -lse2[t]));
                        float ds = p * (dp[kt][t][i] - delta[t]);
                        if (mask && n0 + kt * 16 + grp * 4 + i >= see[t]) ds = 0.f;
                        s[kt][t][i] = ds;
                    }
                df[t] = acc_frag<T>(s[0][t], s[1][t]);      // one rounding of dS to T, as of P
            }
#pragma unroll
            for (int d = 0; d < CD; ++d) {
                const auto kf = col_frag<T, LD>(sk, 0, d * 16);
#pragma unroll
                for (int t = 0; t < NT; ++t) dq[d][t] = mma16(kf, df[t], dq[d][t]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + t * 16 + (lane & 15);
        if (r >= nrow) continue;
        T* p = (T*)a.dq + ((long long)(q0 + tok[t]) * a.heads + kvh * a.group + hd[t]) * a.dim;
#pragma unroll
        for (int d = 0; d < CD; ++d)
            if (d * 16 + grp * 4 < a.dim) store4<T>(p + d * 16 + grp * 4, dq[d][t] * a.scale);
    }
}

// dK, dV: keys in registers, rows (Q and dO) staged 32 at a time.  Here S = Q K^T, so a key is a column of every accumulator,
// and P and dS are again the B operands as they come (dV^T = dO^T P, dK^T = Q^T dS).
template <typename T, int DP, int NW, int NT>
__global__ __launch_bounds__(NW * 64) void dkv_kernel(const AttnArgs a) {
    constexpr int NTHR = NW * 64, BK = NW * NT * 16, BR = 32, LD = DP + Tile<T>::PAD, CK = DP / 32, CD = DP / 16;
    __shared__ __attribute__((aligned(16))) T sq[BR * LD];
    __shared__ __attribute__((aligned(16))) T sg[BR * LD];
    __shared__ __attribute__((aligned(16))) float slse[BR];
    __shared__ __attribute__((aligned(16))) float sdel[BR];
    __shared__ int ssee[BR];
    __shared__ int sh[16];
    const int kvh = blockIdx.x % a.kv_heads, bid = blockIdx.x / a.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 4;
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
    const int nrow = nq * a.group, off = nk - nq;
    const int key0 = w.tile * BK + wave * NT * 16;
    const T* qb = (const T*)a.q + (long long)q0 * a.q_tok + (long long)kvh * a.group * a.q_head;
    const T* gb = (const T*)a.dout + (long long)q0 * a.g_tok + (long long)kvh * a.group * a.g_head;
    const T* kb = (const T*)a.k + (long long)k0 * a.k_tok + (long long)kvh * a.k_head;
    const T* vb = (const T*)a.v + (long long)k0 * a.v_tok + (long long)kvh * a.v_head;
    typename Vec<T>::x8 kf[NT][CK], vf[NT][CK];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int key = key0 + t * 16 + (lane & 15);
        const long long kk = min(key, nk - 1);
#pragma unroll
        for (int c = 0; c < CK; ++c) {
            kf[t][c] = global_frag<T>(kb + kk * a.k_tok, c, a.dim, key < nk);
            vf[t][c] = global_frag<T>(vb + kk * a.v_tok, c, a.dim, key < nk);
        }
    }
    f32x4 dk[CD][NT], dv[CD][NT];
#pragma unroll
    for (int d = 0; d < CD; ++d)
#pragma unroll
        for (int t = 0; t < NT; ++t) dk[d][t] = dv[d][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float c2 = a.scale * LOG2E;
    // the first row that sees the workgroup's first key
    const int first = a.causal ? min(max(w.tile * BK - off, 0), nq) * a.group / BR * BR : 0;
    Stage<T, BR, DP, NTHR> stq, stg;
    float rl = 0.f, rd = 0.f;
    int rs = 0;
    auto fetch = [&](int r0) __attribute__((always_inline)) {
        stq.load_rows(qb, a.q_tok, a.q_head, a.group, r0, nrow, a.dim);
        stg.load_rows(gb, a.g_tok, a.g_head, a.group, r0, nrow, a.dim);
        if (threadIdx.x < BR) {
            const int r = r0 + threadIdx.x, rr = min(r, nrow - 1), t = rr / a.group;
            const long long at = (long long)(q0 + t) * a.heads + kvh * a.group + (rr - t * a.group);
            rl = a.lse[at] * LOG2E;
            rd = a.delta[at];
            rs = r < nrow ? (a.causal ? min(nk, max(t + off + 1, 0)) : nk) : 0;
        }
    };
    if (first < nrow) fetch(first);
    for (int r0 = first; r0 < nrow; r0 += BR) {
        stq.store(sq);
        stg.store(sg);
        if (threadIdx.x < BR) { slse[threadIdx.x] = rl; sdel[threadIdx.x] = rd; ssee[threadIdx.x] = rs; }
        __syncthreads();
        if (r0 + BR < nrow) fetch(r0 + BR);
        if (key0 < ssee[BR - 1] || r0 + BR > nrow) {        // the last row of the step sees most
            f32x4 s[2][NT], dp[2][NT];
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
                for (int t = 0; t < NT; ++t) s[rt][t] = dp[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CK; ++c) {
                    const auto qf = row_frag<T, LD>(sq, rt * 16, c);
                    const auto gf = row_frag<T, LD>(sg, rt * 16, c);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        s[rt][t] = mma16(qf, kf[t][c], s[rt][t]);
                        dp[rt][t] = mma16(gf, vf[t][c], dp[rt][t]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = rt * 16 + grp * 4 + i;
                    const float lse2 = slse[r], del = sdel[r];
                    const int see = ssee[r];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float p = __builtin_amdgcn_exp2f(fmaf(s[rt][t][i], c2, -lse2));
                        float ds = p * (dp[rt][t][i] - del);
                        if (key0 + t * 16 + (lane & 15) >= see) p = ds = 0.f;
                        s[rt][t][i] = p;
                        dp[rt][t][i] = ds;
                    }
                }
            }
            typename Vec<T>::x8 pf[NT], df[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) { pf[t] = acc_frag<T>(s[0][t], s[1][t]); df[t] = acc_frag<T>(dp[0][t], dp[1][t]); }
#pragma unroll
            for (int d = 0; d < CD; ++d) {
                const auto gt = col_frag<T, LD>(sg, 0, d * 16);
                const auto qt = col_frag<T, LD>(sq, 0, d * 16);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    dv[d][t] = mma16(gt, pf[t], dv[d][t]);
                    dk[d][t] = mma16(qt, df[t], dk[d][t]);
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int key = key0 + t * 16 + (lane & 15);
        if (key >= nk) continue;
        const long long at = ((long long)(k0 + key) * a.kv_heads + kvh) * a.dim;
#pragma unroll
        for (int d = 0; d < CD; ++d)
            if (d * 16 + grp * 4 < a.dim) {
                store4<T>((T*)a.dk + at + d * 16 + grp * 4, dk[d][t] * a.scale);
                store4<T>((T*)a.dv + at + d * 16 + grp * 4, dv[d][t]);
            }
    }
}

// ------------------------------------------------------------------------------------------------ host
// workgroups: no more tiles than rows / BM full ones and one partial one a sequence, and one for the rows behind them, each for
// every key head (the fastest index: neighbours in time work on the same few heads of an XCD, whose L2 then holds their keys)
inline unsigned blocks_for(const AttnArgs& a, long long rows, int bm) { return (unsigned)((rows / bm + a.seqs + 1) * a.kv_heads); }

template <typename T, int DP, int NW, int NT>
int launch_fwd(const AttnArgs& a, hipStream_t st) {
    const dim3 grid(blocks_for(a, (long long)a.tokens_q * a.group, NW * NT * 16), a.splits);
    hipLaunchKernelGGL((fwd_kernel<T, DP, NW, NT>), grid, dim3(NW * 64), 0, st, a);
    if (a.splits > 1) {
        const int rpb = 256 / (a.dim / 4);
        const long long rows = (long long)a.tokens_q * a.heads;
        hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)((rows + rpb - 1) / rpb)), dim3(256), 0, st, a);
    }
    return launch_status("attention_packed_fwd");
}

template <typename T, int DP, int NW, int NT>
int launch_dq(const AttnArgs& a, hipStream_t st) {
    const dim3 grid(blocks_for(a, (long long)a.tokens_q * a.group, NW * NT * 16));
    hipLaunchKernelGGL((dq_kernel<T, DP, NW, NT>), grid, dim3(NW * 64), 0, st, a);
    return launch_status("attention_packed_bwd");
}

template <typename T, int DP, int NW, int NT>
int launch_dkv(const AttnArgs& a, hipStream_t st) {
    const dim3 grid(blocks_for(a, a.tokens_k, NW * NT * 16));
    hipLaunchKernelGGL((dkv_kernel<T, DP, NW, NT>), grid, dim3(NW * 64), 0, st, a);
    return launch_status("attention_packed_bwd");
}

}  // namespace attn
}  // namespace icap
