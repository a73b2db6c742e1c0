// Attention over packed sequences (no padding: sequence b owns rows cu[b] .. cu[b + 1] of the packed tensors), forward and
// gradients, for one element type T.
//   S = scale q k^T (keys after a query's place hidden when causal, places aligned at the sequences' ENDS), P = softmax(S), O = P V
//   dV = P^T dO,  dS = P (dO V^T - rowsum(dO O)),  dQ = scale dS K,  dK = scale dS^T Q
// Query heads that share a key head are rows of one matrix: row r is (token r / group, head r % group).  A key is read once
// for the whole group, and dK / dV sum over it inside one workgroup, in a fixed order, without atomics.
// Tiles are consecutive rows (keys, for dK and dV) of the packed tensors, WHATEVER sequences they belong to: every row knows
// the range of keys it sees (every key the range of rows that see it), a tile walks over the union of its rows' ranges, and
// the rest is masked.  Short captions fill tiles together, single tokens of many texts too, and no tile is empty.
//
// One pass over the keys with a running maximum and sum.  The products are formed transposed (S^T = K Q^T, O^T = V^T P^T) on
// 32 x 32 x 16 matrix instructions, so that a query is a column (lane % 32) of every accumulator: its maximum, sum and
// rescaling stay in the lane, and the eight values a lane half holds of 16 accumulator rows are the B operand of the next product as
// they come (V^T is read in the same order of the contraction).  Rows that see no key get zeros (and a log-sum of -inf).
//
// Tiles are multiplied whole, so that a tile's products meet places that its rows do not see: those get the weight zero, and a row whose
// result is not finite is formed once more from what it sees alone ("values that are not finite" below).
//
// What bounds it: at dim 128 a wave of 32 rows needs per 64 keys 1024 cycles of its SIMD's matrix core and about as many of
// its vector unit (32 exponentials of 16 cycles), and the two overlap only in part: 874 TFLOP/s on six bf16 prompts of up to 8192 tokens
// (366 us; a product of that many operations alone takes 252), matrix cores busy 47 % of the cycles, LDS without conflicts.  About 13 % of
// them are a tail, as the longest text's tiles do not start first (fwd_kernel).  Two waves a SIMD interleave (four-wave workgroups, two a CU: with one of eight waves all were in the same phase, 404 against 383 us on
// those prompts), the scores of the next step are formed beside the exponentials of this one (383 -> 353 us), and nothing
// else stays in the loop:
//   * tiles go global -> LDS without registers, double-buffered, one barrier a step;
//   * LDS rows are not padded (the direct loads write linearly) but permuted in 16-byte slots by swizzle(), which spreads the
//     rows of a fragment read and the 4 rows of a transposing read over different banks;
//   * the running maximum is only followed when it grows by more than 2^8 (weights stay below 256, sums in fp32, so nothing
//     is lost), which leaves the accumulators alone in almost every step.
// Backward, 8 bf16 sequences of up to 2048 tokens, dim 64: dK and dV 117, dQ 78, forward 60 us; the steps of the longest sequence's first
// keys, one after another, are what they last.  Short texts (fp32 captions of up to 58 tokens: forward 34, dQ 44, dK and dV 49 us) are
// bound by places of other texts in their tiles: 6.1 times the pairs that are seen are multiplied in the forward pass, 4.6 (dQ) and
// 4.1 (dK, dV) times in the backward pass.
#pragma once
#include "packed.hpp"

namespace icap {
namespace attn {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// acc[32 x 32] += A[32 x 16] B[16 x 32]: a lane brings eight values of A's row and of B's column lane % 32; acc: column lane % 32,
// register e is row acc_row(e) + 4 (lane / 32).  fp32: slot j of all lanes is one 2-deep product.
__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ constexpr int acc_row(int e) { return (e & 3) + 8 * (e >> 2); }

__device__ __forceinline__ f32x16 zeros16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}

__device__ __forceinline__ int cut(int v, int lo, int hi) { return min(max(v, lo), hi); }

// ------------------------------------------------------------------------------------------------ tiles in LDS
// permutation of a row's 16-byte slots.  A 256-byte line of the 64 banks holds one row of 256 bytes (half of one of 512), two of 128 or
// four of 64.  A fragment read takes one slot of 16 rows at a time, which have to lie in 16 places of the line; a transposing read
// takes 64 bytes of four consecutive rows, so those differ in the upper bits.  (With 8 places instead of 16, half of the LDS
// cycles were conflicts.)
template <typename T, int DP>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (sizeof(T) == 4) return DP == 32 ? (row >> 1) & 7 : ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3);
    else if constexpr (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (DP == 64) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
}

// the values of a lane and of lane ^ 32, without the LDS: the swap hands every lane both halves'
__device__ __forceinline__ f32x2 both_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f32x2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// [ROWS][DP] values, global -> LDS
template <typename T, int ROWS, int DP, int NTHR>
struct Direct {
    static constexpr int EPC = 16 / sizeof(T), CH = DP / EPC, PIECES = ROWS * CH, N = PIECES < NTHR ? 1 : PIECES / NTHR;
    static_assert(PIECES < NTHR ? PIECES % 64 == 0 : PIECES % NTHR == 0, "whole passes, or whole waves of one");
    int row[N], col[N];
    __device__ __forceinline__ void init(int dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + i * NTHR;
            row[i] = c / CH;
            const int s = ((c % CH) ^ swizzle<T, DP>(row[i])) * EPC;
            col[i] = s < dim ? s : 0;           // columns behind dim meet zeros of the other operand
        }
    }
    __device__ __forceinline__ void put(const T* p, int i, T* lds) const {
        if (PIECES < NTHR && threadIdx.x >= PIECES) return;         // a short tile does not need every wave
        __builtin_amdgcn_global_load_lds(p, (__attribute__((address_space(3))) void*)(lds + ((threadIdx.x >> 6) * 64 + i * NTHR) * EPC), 16, 0, 0);
    }
    // rows first .. of `valid` (>= 1) rows that are `stride` apart; rows outside repeat the nearest one (they are masked)
    __device__ __forceinline__ void load(const T* src, long long stride, int first, int valid, T* lds) const {
        const T* p = src + first * stride;
#pragma unroll
        for (int i = 0; i < N; ++i) put(p + (cut(row[i], -first, valid - 1 - first) * (int)stride + col[i]), i, lds);
    }
    // rows that are (token, head of the group) pairs
    __device__ __forceinline__ void load_rows(const T* src, int tok, int head, int group, int row0, int end, T* lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = min(row0 + row[i], end - 1), t = r / group;
            put(src + (long long)t * tok + ((r - t * group) * head + col[i]), i, lds);
        }
    }
};

// everything this wave asked for (in LDS, too) has landed, and every wave is here
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// fragment whose matrix rows are tile rows: row row0 + lane % 32, columns 16 kk + 8 (lane / 32) .. + 7
template <typename T, int DP>
__device__ __forceinline__ typename Vec<T>::x8 row_frag(const T* lds, int row0, int kk) {
    const int lane = threadIdx.x & 63, r = lane & 31, lh = lane >> 5, f = swizzle<T, DP>(r);
    const T* p = lds + (row0 + r) * DP;
    if constexpr (sizeof(T) == 2) return *reinterpret_cast<const typename Vec<T>::x8*>(p + ((kk * 2 + lh) ^ f) * 8);
    else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(p + ((kk * 4 + lh * 2) ^ f) * 4), hi = *reinterpret_cast<const f32x4*>(p + ((kk * 4 + lh * 2 + 1) ^ f) * 4);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// transposed: matrix row = tile column col0 + lane % 32; the contraction runs over 16 tile rows in the order of an accumulator's
// eight registers: rows {0-3, 8-11} + 4 (lane / 32).  16-bit types: the transposing LDS read, which hands lane l of 16 column l of the
// 4 x 16 block that its 16 lanes address.
template <typename T, int DP>
__device__ __forceinline__ typename Vec<T>::x8 col_frag(const T* lds, int row0, int col0) {
    const int lane = threadIdx.x & 63, lh = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        const int l = lane & 15, half = (lane >> 4) & 1, r = 4 * lh + (l >> 2), slot = (col0 >> 3) + half * 2 + ((l & 3) >> 1);
        const int f = slot ^ swizzle<T, DP>(r);                 // eight rows further the permutation differs by 2
        const T* p = lds + (row0 + r) * DP + f * 8 + (l & 1) * 4;
        const T* q = lds + (row0 + r + 8) * DP + (f ^ 2) * 8 + (l & 1) * 4;
        typedef __attribute__((address_space(3))) i16x4* lds_ptr;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(q));
        typedef short i16x8 __attribute__((ext_vector_type(8)));
        const i16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(typename Vec<T>::x8, both);
    } else {
        const int col = col0 + (lane & 31);
        typename Vec<T>::x8 f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = (j & 3) + 8 * (j >> 2) + 4 * lh;
            f[j] = lds[(row0 + r) * DP + ((col >> 2) ^ swizzle<T, DP>(r)) * 4 + (col & 3)];
        }
        return f;
    }
}

// eight registers of an accumulator (16 of its rows) as an operand: the one rounding of P to a 16-bit type (2^-8 / 2^-11 of
// each value, as much as the result's own rounding: O is up to 1.3 times as far off as a rounding of the exact result; a second
// part would double the product with V; the sum of P itself is taken from the unrounded values)
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 acc_frag(const f32x16& a, int half) {
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = a[half * 8 + e];
    if constexpr (sizeof(T) == 4) return x;
    else return __builtin_convertvector(x, typename Vec<T>::x8);
}

// dS in two parts, high and low (16-bit types; 16 bits and more of each value, of fp16 with the power of two of lower() below): its terms
// differ in sign, so that one rounded part made dQ and dK 1.53 times as far off as rounding the exact results does; two: 1.17 times, the
// rest from O's own rounding in delta.  The second product costs 8 % of a training pass (222 -> 241 us, 8 bf16 sequences of up to 2048 tokens, dim 64) to 19 % (dim 128).
template <typename T>
__device__ __forceinline__ void acc_parts(const f32x16& a, int half, typename Vec<T>::x8& hi, typename Vec<T>::x8& lo) {
    f32x8 x, y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = a[half * 8 + e];
        if constexpr (__is_same(T, __bf16)) y[e] = __uint_as_float(__float_as_uint(x[e]) & 0xffff0000u);
    }
    if constexpr (__is_same(T, __bf16)) {
        hi = __builtin_convertvector(y, typename Vec<T>::x8);
    } else {
        hi = __builtin_convertvector(x, typename Vec<T>::x8);
        y = __builtin_convertvector(hi, f32x8);
    }
    lo = __builtin_convertvector(x - y, typename Vec<T>::x8);
}

// fp16 ends at 2^-24 and at 65504, and dS, a weight times an output gradient, at neither: over 4096 keys and gradients of 1e-3 it is some 2e-6, of
// which the two parts held 5 bits.  So a column's dS (its row's in dQ, its key's in dK) are formed with a power of two, which the
// column's accumulators then have, too.  It starts at 2^40 and is lowered when a value would pass 2^15: the largest so far is at 2^8
// and above (or below 2^-25), and values down to 2^-11 of it have all 22 bits.  Backward pass of 8 fp16 sequences of up to 2048 tokens, dim 64:
// 155 -> 163 us, 16 of 1024, dim 128: 623 -> 707; under a loss scale with which dS passed 65504, and every such row was formed once
// more ("values that are not finite" below), 13.5 ms -> 163 us.
constexpr int LIFT0 = 40;
__device__ __forceinline__ float power_of(int b) { return __uint_as_float((unsigned)(b + 127) << 23); }
// s: dS 2^bits of 16 places
template <int ND>
__device__ __forceinline__ void lower(f32x16& s, int& bits, f32x16 (&acc)[ND]) {
    float most = fabsf(s[0]), other = fabsf(s[8]);
#pragma unroll
    for (int e = 1; e < 8; ++e) { most = fmaxf(most, fabsf(s[e])); other = fmaxf(other, fabsf(s[e + 8])); }
    most = fmaxf(most, other);
    if (__builtin_expect(__any(most > 32768.0f), 0)) {
        const f32x2 halves = both_halves(most);
        most = fmaxf(halves[0], halves[1]);
        // to 2^8 (from 2^127 at most; what is not finite stays that)
        const int by = most > 32768.0f ? max(8 - ((int)(__float_as_uint(most) >> 23) - 127), -100 - bits) : 0;
        const float f = power_of(by);
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= f;
        s *= f;
        bits += by;
    }
}

// fragment of a row in memory: columns 16 kk + 8 (lane / 32) .. + 7, zeros from dim on and when !ok (p stays readable)
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 global_frag(const T* row, int kk, int dim, bool ok) {
    const int col = kk * 16 + ((threadIdx.x & 63) >> 5) * 8;
    typename Vec<T>::x8 f = *reinterpret_cast<const typename Vec<T>::x8*>(row + (col < dim ? col : 0));
    if (!(ok && col < dim)) f = typename Vec<T>::x8{};
    return f;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
    else *reinterpret_cast<typename Vec<T>::x4*>(p) = __builtin_convertvector(v, typename Vec<T>::x4);
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

// ------------------------------------------------------------------------------------------------ who sees whom
struct Span { int lo, hi; };

// the last sequences that begin at or before places x and y (x <= y), by all 64 lanes of a wave: 64 offsets at a time, two loads for up
// to 4096 sequences
__device__ __forceinline__ void find_two(const int* cu, int seqs, int x, int y, int& sx, int& sy) {
    const int lane = threadIdx.x & 63;
    int lx = 0, nx = seqs, ly = 0, ny = seqs;
    while (nx > 1 || ny > 1) {
        const int ax = (nx + 63) >> 6, ay = (ny + 63) >> 6;
        const bool ox = lane * ax < nx && cu[lx + lane * ax] <= x, oy = lane * ay < ny && cu[ly + lane * ay] <= y;
        const int px = max(__popcll(__ballot(ox)) - 1, 0) * ax, py = max(__popcll(__ballot(oy)) - 1, 0) * ay;
        lx += px;
        nx = min(ax, nx - px);
        ly += py;
        ny = min(ay, ny - py);
    }
    sx = __builtin_amdgcn_readfirstlane(lx);
    sy = __builtin_amdgcn_readfirstlane(ly);
}
// the same for a lane of its own, between sequences a and b
__device__ __forceinline__ int find_between(const int* cu, int x, int a, int b) {
    while (a < b) {
        const int mid = (a + b + 1) >> 1;
        if (cu[mid] <= x) a = mid; else b = mid - 1;
    }
    return a;
}

// The keys that a token sees, and the rows that see a key, from the offsets of sequence s (which may be wrong: they are cut off at the
// tensors' ends, and a place outside its sequence sees nothing, so nothing outside is read or written)
struct Edge { int q0, q1, k0, k1; };
__device__ __forceinline__ Edge edge_of(const AttnArgs& a, int s) {
    Edge e;
    e.q0 = cut(a.cu_q[s], 0, a.tokens_q);
    e.q1 = cut(a.cu_q[s + 1], e.q0, a.tokens_q);
    e.k0 = cut(a.cu_k[s], 0, a.tokens_k);
    e.k1 = cut(a.cu_k[s + 1], e.k0, a.tokens_k);
    return e;
}
__device__ __forceinline__ Span keys_of(const AttnArgs& a, const Edge& e, int t) {
    if (t < e.q0 || t >= e.q1) return {e.k0, e.k0};
    return {e.k0, a.causal ? cut(e.k1 - (e.q1 - 1 - t), e.k0, e.k1) : e.k1};
}
__device__ __forceinline__ Span rows_of(const AttnArgs& a, const Edge& e, int j) {
    if (j < e.k0 || j >= e.k1) return {e.q0 * a.group, e.q0 * a.group};
    return {(a.causal ? cut(e.q1 - (e.k1 - j), e.q0, e.q1) : e.q0) * a.group, e.q1 * a.group};
}

// What the lanes of a wave see together: anything in [some.lo, some.hi), everything in [all.lo, all.hi)
__device__ __forceinline__ int wave_min_i(int v) {
    v = min(v, dpp_i<DPP_QUAD_SWAP1>(v));
    v = min(v, dpp_i<DPP_QUAD_SWAP2>(v));
    v = min(v, dpp_i<DPP_HALF_MIRROR>(v));
    v = min(v, dpp_i<DPP_ROW_MIRROR>(v));
    return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)), min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
struct Sight { Span mine, some, all; };
__device__ __forceinline__ Sight sight_of(Span s) {
    const bool none = s.lo >= s.hi;
    Sight w;
    w.mine = s;
    w.some = {wave_min_i(none ? 0x7fffffff : s.lo), -wave_min_i(none ? 0x7fffffff : -s.hi)};
    w.all = {-wave_min_i(-s.lo), wave_min_i(s.hi)};
    if (w.some.lo == 0x7fffffff) w.some = {0, 0};
    return w;
}

// A tile of `rows` rows (token, head) from row0: the keys that any of them sees, and what this lane's row sees
template <int ROWS>
__device__ __forceinline__ Span tile_keys(const AttnArgs& a, int row0, int row, Sight& sight) {
    const int total = a.tokens_q * a.group, end = cut(a.cu_q[a.seqs], 0, a.tokens_q);
    const int t0 = row0 / a.group, t1 = min(min(row0 + ROWS, total) - 1, end * a.group - 1) / a.group;
    if (t0 >= end) { sight = sight_of({0, 0}); return {0, 0}; }          // behind the last sequence
    int s0, s1;
    find_two(a.cu_q, a.seqs, t0, t1, s0, s1);
    const int t = min(row, total - 1) / a.group;
    const Edge e = edge_of(a, find_between(a.cu_q, min(t, t1), s0, s1));
    sight = sight_of(row < total ? keys_of(a, e, t) : Span{e.k0, e.k0});
    const Edge e0 = edge_of(a, s0), e1 = edge_of(a, s1);
    return {e0.k0, keys_of(a, e1, t1).hi};
}
// A tile of keys from key0: the rows that see any of them, and the ones that see this lane's key
template <int KEYS>
__device__ __forceinline__ Span tile_rows(const AttnArgs& a, int key0, int key, Sight& sight) {
    const int end = cut(a.cu_k[a.seqs], 0, a.tokens_k);
    const int j1 = min(key0 + KEYS, end) - 1;
    if (key0 >= end) { sight = sight_of({0, 0}); return {0, 0}; }
    int s0, s1;
    find_two(a.cu_k, a.seqs, key0, j1, s0, s1);
    const Edge e = edge_of(a, find_between(a.cu_k, min(key, j1), s0, s1));
    sight = sight_of(key < end ? rows_of(a, e, key) : Span{0, 0});
    const Edge e0 = edge_of(a, s0), e1 = edge_of(a, s1);
    return {rows_of(a, e0, key0).lo, rows_of(a, e1, j1).hi};
}

// ------------------------------------------------------------------------------------------------ values that are not finite
// What a row does not see has the weight zero, but zero times an infinity or a NaN is not zero, and a tile's products meet the keys of
// all its rows.  So a row (key) whose results are not all finite is formed once more, by its two lanes, from what it sees and nothing
// else.  Slow, and not reached by finite tensors whose scores, weights, dO V^T and sums are finite in fp32.
template <int ND>
__device__ __forceinline__ bool finite_row(const f32x16 (&x)[ND]) {
    float z = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) z = fmaf(x[d][e], 0.f, z);
    z += __shfl_xor(z, 32);
    return z == 0.f;
}
// x . y, half of the columns by each of the two lanes that share a row
template <typename T>
__device__ __forceinline__ float pair_dot(const T* x, const T* y, int dim) {
    float s = 0.f;
    for (int c = ((threadIdx.x & 63) >> 5) * 8; c < dim; c += 16) {
        const auto a = *reinterpret_cast<const typename Vec<T>::x8*>(x + c), b = *reinterpret_cast<const typename Vec<T>::x8*>(y + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf((float)a[e], (float)b[e], s);
    }
    return s + __shfl_xor(s, 32);
}
// a lane's columns of a result row (store16's) += w x
template <typename T, int ND>
__device__ __forceinline__ void add_row(f32x16 (&acc)[ND], float w, const T* x, int dim) {
    const int lh = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = d * 32 + 8 * g + 4 * lh;
            if (c < dim) {
                const auto v = *reinterpret_cast<const typename Vec<T>::x4*>(x + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[d][4 * g + i] = fmaf(w, (float)v[i], acc[d][4 * g + i]);
            }
        }
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T> constexpr int step_keys() { return sizeof(T) == 4 ? 32 : 64; }       // keys (rows) staged at a time

template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, DP == 128 && (NW < 4 || sizeof(T) == 4) ? 1 : 2) void fwd_kernel(const AttnArgs a) {
    constexpr int NTHR = NW * 64, BM = NW * 32, BN = step_keys<T>(), NS = BN / 32, KK = DP / 16, ND = DP / 32;
    __shared__ __attribute__((aligned(1024))) T sk[2][BN * DP];
    __shared__ __attribute__((aligned(1024))) T sv[2][BN * DP];
    const int kvh = blockIdx.x % a.kv_heads, tiles = gridDim.x / a.kv_heads, lane = threadIdx.x & 63, lh = lane >> 5;
    // causal: later rows of a sequence see more keys and start first.  Sequences go in the order they are given, the last one first (507,
    // 112, 4, 8192, 301 and 3254 tokens: 187 steps one after another, 162 if the longest tiles started first)
    const int tile = a.causal ? tiles - 1 - (int)(blockIdx.x / a.kv_heads) : blockIdx.x / a.kv_heads;
    const int row0 = tile * BM, row = row0 + (threadIdx.x >> 6) * 32 + (lane & 31), total = a.tokens_q * a.group;
    const int tok = min(row, total - 1) / a.group, head = kvh * a.group + min(row, total - 1) - tok * a.group;
    Sight me;
    Span keys = tile_keys<BM>(a, row0, row, me);
    if (a.splits > 1) {             // the part of the keys that this workgroup takes: whole steps, at least two of them
        const int steps = (keys.hi - keys.lo + BN - 1) / BN, per = max((steps + a.splits - 1) / a.splits, 2) * BN;
        keys.lo = min(keys.lo + (int)blockIdx.y * per, keys.hi);
        keys.hi = min(keys.lo + per, keys.hi);
    }
    const T* qp = (const T*)a.q + (long long)tok * a.q_tok + (long long)head * a.q_head;
    // places from here on are counted from the tile's first key
    const T* kb = (const T*)a.k + (long long)keys.lo * a.k_tok + (long long)kvh * a.k_head;
    const T* vb = (const T*)a.v + (long long)keys.lo * a.v_tok + (long long)kvh * a.v_head;
    const int nk = keys.hi - keys.lo, full_lo = me.all.lo - keys.lo, full_hi = me.all.hi - keys.lo;
    const int see_lo = me.mine.lo - keys.lo - 4 * lh, see_hi = me.mine.hi - keys.lo - 4 * lh;
    typename Vec<T>::x8 qf[KK];
#pragma unroll
    for (int c = 0; c < KK; ++c) qf[c] = global_frag<T>(qp, c, a.dim, row < total);

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = zeros16();
    float m = -INFINITY, l = 0.f;
    // fp16 ends at 2^-24: weights (up to 2^8, see above) are taken 2^7 times, as their sum then is; 11 bits down to 2^-21 of the largest
    constexpr float P_BITS = __is_same(T, _Float16) ? 7.0f : 0.0f;
    const float c2 = a.scale * LOG2E;
    // The scores of the next 32 keys are formed while the exponentials of these run, so K is staged 32 keys ahead of V: a step of
    // V's keys n0 .. n0 + BN goes with K's n0 + 32 .. n0 + BN + 32
    Direct<T, BN, DP, NTHR> dir;
    dir.init(a.dim);
    auto load = [&](int n0, int buf) __attribute__((always_inline)) {
        dir.load(kb, a.k_tok, n0 + 32, nk, sk[buf]);
        dir.load(vb, a.v_tok, n0, nk, sv[buf]);
    };
    auto scores = [&](const T* tile, int row) __attribute__((always_inline)) {
        f32x16 s = zeros16();
#pragma unroll
        for (int c = 0; c < KK; ++c) s = mma32(row_frag<T, DP>(tile, row, c), qf[c], s);
        return s;
    };
    // `now`: scores of the 32 keys from n (rows vr of the V tile); returns those of the next 32 (rows kr of the K tile)
    auto unit = [&](f32x16 now, int n, const T* vt, int vr, const T* kt, int kr) __attribute__((always_inline)) {
        if (n < full_lo || n + 32 > full_hi) {
            const int lo = see_lo - n, hi = see_hi - n;         // against constants: no register a place
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (acc_row(e) < lo || acc_row(e) >= hi) now[e] = -INFINITY;
        }
        float mx = now[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, now[e]);
        const f32x2 halves = both_halves(mx);
        mx = fmaxf(halves[0], halves[1]) * c2;
        if (__any(mx > m + 8.0f)) {
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
        }
        const f32x16 next = scores(kt, kr);
        const float base = (m == -INFINITY ? 0.f : m) - P_BITS;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = __builtin_amdgcn_exp2f(fmaf(now[j * 8 + e], c2, -base));
                now[j * 8 + e] = p;
                sum += p;
            }
            const auto pf = acc_frag<T>(now, j);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = mma32(col_frag<T, DP>(vt, vr + j * 16, d * 32), pf, o[d]);
        }
        l += sum;
        return next;
    };
    if (nk > 0) {
        dir.load(kb, a.k_tok, 32 - BN, nk, sk[1]);              // its last 32 rows are the first keys
        load(0, 0);
        landed();
        f32x16 s = scores(sk[1], BN - 32);
        for (int n0 = 0, buf = 0; n0 < nk; n0 += BN, buf ^= 1) {
            landed();
            if (n0 + BN < nk) load(n0 + BN, buf ^ 1);
#pragma unroll
            for (int u = 0; u < NS; ++u) s = unit(s, n0 + 32 * u, sv[buf], 32 * u, sk[buf], 32 * u);
        }
    }
    float sum = l + __shfl_xor(l, 32);
    m -= P_BITS;
    if (!finite_row(o)) {
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = zeros16();
        m = -INFINITY;
        sum = 0.f;
        for (int j = max(me.mine.lo, keys.lo); j < min(me.mine.hi, keys.hi) && sum == sum; ++j) {       // one NaN in the sum: all is NaN
            const long long at = j - keys.lo;
            const float s = pair_dot(qp, kb + at * a.k_tok, a.dim) * c2, most = fmaxf(m, s), base = most == -INFINITY ? 0.f : most;
            const float alpha = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(s - base);
            sum = fmaf(sum, alpha, p);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
            add_row(o, p, vb + at * a.v_tok, a.dim);
            m = most;
        }
    }
    if (row >= total) return;
    const long long at = (long long)tok * a.heads + head;
    const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);        // no key: zeros; NaN stays
    const float lse = sum > 0.f ? fmaf(m, LN2, logf(sum)) : (sum == 0.f ? -INFINITY : sum);
    if (a.splits > 1) {
        const long long rows = (long long)a.tokens_q * a.heads;
        float* part = a.part + (rows * blockIdx.y + at) * a.dim;
#pragma unroll
        for (int d = 0; d < ND; ++d) store16<float>(part, d * 32, a.dim, o[d], inv);
        if (lh == 0) a.part[rows * a.splits * a.dim + rows * blockIdx.y + at] = lse;
    } else {
#pragma unroll
        for (int d = 0; d < ND; ++d) store16<T>((T*)a.out + at * a.dim, d * 32, a.dim, o[d], inv);
        if (lh == 0 && a.lse) a.lse[at] = lse;
    }
}

// joins the parts of split keys: each is a normalised result with its log-sum (zeros and -inf where its keys are none of this row's).
// dim / 4 threads a row, one wave a workgroup.
template <typename T>
__global__ __launch_bounds__(64) void join_kernel(const AttnArgs a) {
    const int per = a.dim / 4, rpb = 64 / per, i = threadIdx.x / per, d = (threadIdx.x - i * per) * 4;
    const long long rows = (long long)a.tokens_q * a.heads, r = (long long)blockIdx.x * rpb + i;
    if (i >= rpb || r >= rows) return;
    const float* pl = a.part + rows * a.splits * a.dim + r;
    const float* po = a.part + r * a.dim + d;
    float most = -INFINITY;
#pragma unroll 8
    for (int z = 0; z < a.splits; ++z) most = fmaxf(most, pl[rows * z]);
    const float base = most == -INFINITY ? 0.f : most;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll 8
    for (int z = 0; z < a.splits; ++z) {
        const float w = __builtin_amdgcn_exp2f((pl[rows * z] - base) * LOG2E);
        sum += w;
        acc += w * *reinterpret_cast<const f32x4*>(po + rows * a.dim * z);
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

// adds up the accumulators of the G waves that share rows (or keys), in the first of them; at: where a lane's values go in LDS
template <int ND, int G>
__device__ __forceinline__ void join_waves(f32x16 (&x)[ND], float* at, int group) {
#pragma unroll
    for (int g = 1; g < G; ++g) {
        __syncthreads();
        if (group == g) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) at[(d * 16 + e) * 64] = x[d][e];
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[d][e] += at[(d * 16 + e) * 64];
        }
    }
}

// dQ: the forward's shape (rows in registers, keys staged), with dO beside Q and dS in P's place.
// RW waves of 32 rows each, KG times: key groups take every KG-th 32 keys of a step, as the row groups of dK and dV do (one causal
// sequence of 4096 tokens, 16 heads of 64, forward and backward: 329 -> 299 us; sequences of 200 tokens: 160 -> 163)
template <typename T, int DP, int RW, int KG>
__global__ __launch_bounds__(RW * KG * 64, DP == 128 && (RW < 4 || sizeof(T) == 4) ? 1 : 2) void dq_kernel(const AttnArgs a) {
    constexpr int NTHR = RW * KG * 64, BM = RW * 32, BN = KG > 1 ? 32 * KG : step_keys<T>(), NS = BN / 32 / KG, KK = DP / 16, ND = DP / 32;
    __shared__ __attribute__((aligned(1024))) T staged[4][BN * DP];
    static_assert(KG == 1 || sizeof(staged) >= RW * 64 * ND * 16 * 4, "dQ of a key group fits the tiles");
    T (*const sk)[BN * DP] = staged;
    T (*const sv)[BN * DP] = staged + 2;
    const int wave = threadIdx.x >> 6, kg = wave / RW, rw = wave - kg * RW;
    const int kvh = blockIdx.x % a.kv_heads, tiles = gridDim.x / a.kv_heads, lane = threadIdx.x & 63, lh = lane >> 5;
    const int tile = a.causal ? tiles - 1 - (int)(blockIdx.x / a.kv_heads) : blockIdx.x / a.kv_heads;
    const int row0 = tile * BM, row = row0 + rw * 32 + (lane & 31), total = a.tokens_q * a.group;
    const int tok = min(row, total - 1) / a.group, head = kvh * a.group + min(row, total - 1) - tok * a.group;
    const long long at = (long long)tok * a.heads + head;
    Sight me;
    const Span keys = tile_keys<BM>(a, row0, row, me);
    const T* qp = (const T*)a.q + (long long)tok * a.q_tok + (long long)head * a.q_head;
    const T* gp = (const T*)a.dout + (long long)tok * a.g_tok + (long long)head * a.g_head;
    const T* kb = (const T*)a.k + (long long)kvh * a.k_head;
    const T* vb = (const T*)a.v + (long long)kvh * a.v_head;
    Direct<T, BN, DP, NTHR> dir;
    dir.init(a.dim);
    auto load = [&](int n0, int buf) __attribute__((always_inline)) {
        dir.load(kb, a.k_tok, n0, keys.hi, sk[buf]);
        dir.load(vb, a.v_tok, n0, keys.hi, sv[buf]);
    };
    if (keys.lo < keys.hi) load(keys.lo, 0);
    const float lse2 = a.lse[at] * LOG2E, delta = a.delta[at], c2 = a.scale * LOG2E;
    typename Vec<T>::x8 qf[KK], gf[KK];
#pragma unroll
    for (int c = 0; c < KK; ++c) {
        qf[c] = global_frag<T>(qp, c, a.dim, row < total);
        gf[c] = global_frag<T>(gp, c, a.dim, row < total);
    }
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[d] = zeros16();
    int bits = __is_same(T, _Float16) ? LIFT0 : 0;
    int buf = 0;
    for (int n0 = keys.lo; n0 < keys.hi; n0 += BN, buf ^= 1) {
        landed();
        if (n0 + BN < keys.hi) load(n0 + BN, buf ^ 1);
#pragma unroll
        for (int ks = 0; ks < NS; ++ks) {
            const int kt = kg * NS + ks, n1 = n0 + kt * 32;
            if (n1 >= me.some.hi || n1 + 32 <= me.some.lo) continue;
            f32x16 s = zeros16(), dp = zeros16();
#pragma unroll
            for (int c = 0; c < KK; ++c) {
                s = mma32(row_frag<T, DP>(sk[buf], kt * 32, c), qf[c], s);
                dp = mma32(row_frag<T, DP>(sv[buf], kt * 32, c), gf[c], dp);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, (float)bits - lse2)) * (dp[e] - delta);
            if (n1 < me.all.lo || n1 + 32 > me.all.hi) {
                const int lo = me.mine.lo - n1 - 4 * lh, hi = me.mine.hi - n1 - 4 * lh;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (acc_row(e) < lo || acc_row(e) >= hi) s[e] = 0.f;
            }
            if constexpr (__is_same(T, _Float16)) lower(s, bits, dq);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if constexpr (sizeof(T) == 4) {
                    const auto df = acc_frag<T>(s, j);
#pragma unroll
                    for (int d = 0; d < ND; ++d) dq[d] = mma32(col_frag<T, DP>(sk[buf], kt * 32 + j * 16, d * 32), df, dq[d]);
                } else {
                    typename Vec<T>::x8 hi, lo;
                    acc_parts<T>(s, j, hi, lo);
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const auto kf = col_frag<T, DP>(sk[buf], kt * 32 + j * 16, d * 32);
                        dq[d] = mma32(kf, lo, mma32(kf, hi, dq[d]));
                    }
                }
            }
        }
    }
    if constexpr (__is_same(T, _Float16)) {
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[d] *= power_of(-bits);
    }
    if constexpr (KG > 1) {
        join_waves<ND, KG>(dq, reinterpret_cast<float*>(staged) + rw * (64 * ND * 16) + lane, kg);
        if (kg > 0) return;
    }
    if (!finite_row(dq)) {
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[d] = zeros16();
        float ds = 0.f;
        for (int j = me.mine.lo; j < me.mine.hi && ds == ds; ++j) {
            const T* kp = kb + (long long)j * a.k_tok;
            const float p = __builtin_amdgcn_exp2f(fmaf(pair_dot(qp, kp, a.dim), c2, -lse2));
            ds = p * (pair_dot(gp, vb + (long long)j * a.v_tok, a.dim) - delta);
            add_row(dq, ds, kp, a.dim);
        }
    }
    if (row >= total) return;
#pragma unroll
    for (int d = 0; d < ND; ++d) store16<T>((T*)a.dq + at * a.dim, d * 32, a.dim, dq[d], a.scale);
}

// dK, dV: keys in registers, rows (Q and dO) staged.  Here S = Q K^T, so a key is a column of every accumulator, and P and dS are again
// the B operands as they come (dV^T = dO^T P, dK^T = Q^T dS).
// KW waves of 32 keys each, RG times: the row groups take every RG-th 32 rows and are added up in LDS at the end.  The first keys of
// a long causal sequence meet all its rows, and that chain of steps - not the sum of the work - is what a launch of few sequences
// lasts (167 -> 109 us with two groups, before dS had two parts, 8 bf16 sequences of up to 2048 tokens, dim 64).
// fp16: P 2^14 is rounded, which keeps 11 bits of a weight down to 2^-28 (of P itself down to 2^-14: keys that are hardly seen by many rows lost
// their dV, 170 times its bound at weights of 1e-8); the factor comes with the row's log-sum and leaves after the loop.
template <typename T, int DP, int KW, int RG>
__global__ __launch_bounds__(KW * RG * 64, DP == 128 ? 1 : 2) void dkv_kernel(const AttnArgs a) {
    constexpr int NTHR = KW * RG * 64, BK = KW * 32, BR = 32 * RG, KK = DP / 16, ND = DP / 32;
    constexpr float P_BITS = __is_same(T, _Float16) ? 14.0f : 0.0f;
    __shared__ __attribute__((aligned(1024))) T tiles[4][BR * DP];
    static_assert(RG == 1 || sizeof(tiles) >= KW * 64 * ND * 16 * 4, "one of dK, dV of a row group fits the tiles");
    T (*const sq)[BR * DP] = tiles;
    T (*const sg)[BR * DP] = tiles + 2;
    __shared__ __attribute__((aligned(16))) float srow[2][2][BR];       // lse, delta
    const int kvh = blockIdx.x % a.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lh = lane >> 5;
    const int rg = wave / KW, kw = wave - rg * KW, mine = rg * 32;      // this wave's rows of a step begin at `mine`
    const int key0 = (int)(blockIdx.x / a.kv_heads) * BK, key = key0 + kw * 32 + (lane & 31);
    Sight me;
    const Span rows = tile_rows<BK>(a, key0, key, me);
    const T* qb = (const T*)a.q + (long long)kvh * a.group * a.q_head;
    const T* gb = (const T*)a.dout + (long long)kvh * a.group * a.g_head;
    Direct<T, BR, DP, NTHR> dir;
    dir.init(a.dim);
    auto fetch = [&](int r0, int buf) __attribute__((always_inline)) {
        dir.load_rows(qb, (int)a.q_tok, (int)a.q_head, a.group, r0, rows.hi, sq[buf]);
        dir.load_rows(gb, (int)a.g_tok, (int)a.g_head, a.group, r0, rows.hi, sg[buf]);
        if (threadIdx.x < BR) {
            const int r = min(r0 + (int)threadIdx.x, rows.hi - 1), t = r / a.group;
            const long long at = (long long)t * a.heads + kvh * a.group + (r - t * a.group);
            srow[buf][0][threadIdx.x] = a.lse[at] * LOG2E - P_BITS;
            srow[buf][1][threadIdx.x] = a.delta[at];
        }
    };
    if (rows.lo < rows.hi) fetch(rows.lo, 0);
    typename Vec<T>::x8 kf[KK], vf[KK];
    {
        const long long kk = min(key, a.tokens_k - 1);
        const T* kp = (const T*)a.k + kk * a.k_tok + (long long)kvh * a.k_head;
        const T* vp = (const T*)a.v + kk * a.v_tok + (long long)kvh * a.v_head;
#pragma unroll
        for (int c = 0; c < KK; ++c) {
            kf[c] = global_frag<T>(kp, c, a.dim, key < a.tokens_k);
            vf[c] = global_frag<T>(vp, c, a.dim, key < a.tokens_k);
        }
    }
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zeros16();
    const float c2 = a.scale * LOG2E;
    int bits = __is_same(T, _Float16) ? LIFT0 : 0;
    int buf = 0;
    for (int r0 = rows.lo; r0 < rows.hi; r0 += BR, buf ^= 1) {
        landed();
        if (r0 + BR < rows.hi) fetch(r0 + BR, buf ^ 1);
        const int r1 = r0 + mine;
        if (r1 >= me.some.hi || r1 + 32 <= me.some.lo) continue;
        f32x16 s = zeros16(), dp = zeros16();
#pragma unroll
        for (int c = 0; c < KK; ++c) {
            s = mma32(row_frag<T, DP>(sq[buf], mine, c), kf[c], s);
            dp = mma32(row_frag<T, DP>(sg[buf], mine, c), vf[c], dp);
        }
        const float factor = power_of(bits);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(&srow[buf][0][mine + 8 * g + 4 * lh]), d4 = *reinterpret_cast<const f32x4*>(&srow[buf][1][mine + 8 * g + 4 * lh]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = 4 * g + i;
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, -l4[i]));
                if constexpr (__is_same(T, _Float16)) dp[e] = s[e] * fmaf(dp[e], factor, -d4[i] * factor);
                else dp[e] = s[e] * (dp[e] - d4[i]);
            }
        }
        if (r1 < me.all.lo || r1 + 32 > me.all.hi) {
            const int lo = me.mine.lo - r1 - 4 * lh, hi = me.mine.hi - r1 - 4 * lh;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (acc_row(e) < lo || acc_row(e) >= hi) s[e] = dp[e] = 0.f;
        }
        if constexpr (__is_same(T, _Float16)) lower(dp, bits, dk);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const auto pf = acc_frag<T>(s, j);
            typename Vec<T>::x8 hi, lo;
            if constexpr (sizeof(T) == 4) hi = acc_frag<T>(dp, j);
            else acc_parts<T>(dp, j, hi, lo);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                dv[d] = mma32(col_frag<T, DP>(sg[buf], mine + j * 16, d * 32), pf, dv[d]);
                const auto qt = col_frag<T, DP>(sq[buf], mine + j * 16, d * 32);
                dk[d] = mma32(qt, hi, dk[d]);
                if constexpr (sizeof(T) == 2) dk[d] = mma32(qt, lo, dk[d]);
            }
        }
    }
    if constexpr (__is_same(T, _Float16)) {
        const float p_factor = __builtin_amdgcn_exp2f(-P_BITS);
        const float factor = power_of(-bits) * p_factor;
#pragma unroll
        for (int d = 0; d < ND; ++d) { dk[d] *= factor; dv[d] *= p_factor; }
    }
    if constexpr (RG > 1) {
        float* at = reinterpret_cast<float*>(tiles) + kw * (64 * ND * 16) + lane;
        join_waves<ND, RG>(dk, at, rg);
        join_waves<ND, RG>(dv, at, rg);
        if (rg > 0) return;
    }
    if (!finite_row(dk) || !finite_row(dv)) {
#pragma unroll
        for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zeros16();
        const long long kk = min(key, a.tokens_k - 1);
        const T* kp = (const T*)a.k + kk * a.k_tok + (long long)kvh * a.k_head;
        const T* vp = (const T*)a.v + kk * a.v_tok + (long long)kvh * a.v_head;
        float p = 0.f;
        for (int r = me.mine.lo; r < me.mine.hi && p == p; ++r) {
            const int t = r / a.group, h = r - t * a.group;
            const T* qp = qb + t * a.q_tok + h * a.q_head;
            const T* gp = gb + t * a.g_tok + h * a.g_head;
            const long long at = (long long)t * a.heads + kvh * a.group + h;
            p = __builtin_amdgcn_exp2f(fmaf(pair_dot(qp, kp, a.dim), c2, -a.lse[at] * LOG2E));
            add_row(dv, p, gp, a.dim);
            add_row(dk, p * (pair_dot(gp, vp, a.dim) - a.delta[at]), qp, a.dim);
        }
    }
    if (key >= a.tokens_k) return;
    const long long at = ((long long)key * a.kv_heads + kvh) * a.dim;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        store16<T>((T*)a.dk + at, d * 32, a.dim, dk[d], a.scale);
        store16<T>((T*)a.dv + at, d * 32, a.dim, dv[d], 1.0f);
    }
}

// ------------------------------------------------------------------------------------------------ host
// one workgroup for every tile of `per` rows and every key head (the fastest index: neighbours in time work on the few heads of an XCD,
// whose L2 then holds their keys)
inline unsigned blocks_for(const AttnArgs& a, long long rows, int per) { return (unsigned)((rows + per - 1) / per * a.kv_heads); }

template <typename T, int DP, int NW>
int launch_fwd(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((fwd_kernel<T, DP, NW>), dim3(blocks_for(a, (long long)a.tokens_q * a.group, NW * 32), a.splits), dim3(NW * 64), 0, st, a);
    if (a.splits > 1) {
        const int rpb = 64 / (a.dim / 4);
        hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(((long long)a.tokens_q * a.heads + rpb - 1) / rpb)), dim3(64), 0, st, a);
    }
    return launch_status("attention_packed_fwd");
}
template <typename T, int DP, int RW, int KG>
void launch_dq(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((dq_kernel<T, DP, RW, KG>), dim3(blocks_for(a, (long long)a.tokens_q * a.group, RW * 32)), dim3(RW * KG * 64), 0, st, a);
}
template <typename T, int DP, int KW, int RG>
void launch_dkv(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((dkv_kernel<T, DP, KW, RG>), dim3(blocks_for(a, a.tokens_k, KW * 32)), dim3(KW * RG * 64), 0, st, a);
}

// Waves a workgroup: four where the average sequence fills them, since they share each staged tile (two / four: bf16 prompts of up to 8192
// tokens 574 / 361 us), two otherwise (fp32 captions of up to 58 tokens, forward and backward, 136 / 148); split keys go with one wave
// (attention_splits in capi.hip: few rows, long caches)
template <typename T, int DP>
int fwd_dim(const AttnArgs& a, hipStream_t st) {
    if (a.splits > 1) return launch_fwd<T, DP, 1>(a, st);
    if ((long long)a.tokens_q * a.group / a.seqs <= 96) return launch_fwd<T, DP, 2>(a, st);
    return launch_fwd<T, DP, 4>(a, st);
}

// Backward: a wave that walks alone over all a sequence's keys (rows) is what a launch lasts, as long as there are fewer workgroups than the
// card takes at once (some 2048 of two waves); then two groups of waves share the walk.  16-bit types, dim 64, alone / shared: 8
// sequences of 512 tokens, 8 heads 79 / 63 us; of up to 2048 324 / 239; but 64 of 200, 16 heads (3200 workgroups) 156 / 172, 16 of 1024 with
// dim 128 (2048) 430 / 478.  Not where a walk is a few steps anyway: fp32 captions of up to 58 tokens 136 / 173.
template <typename T, int DP>
int bwd_dim(const AttnArgs& a, hipStream_t st) {
    const long long all = (long long)a.tokens_q * a.group;
    const bool lengthy = all / a.seqs > 96;
    if (a.tokens_q > 0) {
        if (lengthy && blocks_for(a, all, 64) < 2048) launch_dq<T, DP, 2, 2>(a, st);
        else launch_dq<T, DP, 2, 1>(a, st);
    }
    if (a.tokens_k > 0) {
        if (lengthy && blocks_for(a, a.tokens_k, 64) < 2048) launch_dkv<T, DP, 2, 2>(a, st);
        else launch_dkv<T, DP, 2, 1>(a, st);
    }
    return launch_status("attention_packed_bwd");
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
