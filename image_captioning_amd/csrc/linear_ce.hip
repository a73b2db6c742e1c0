// Softmax cross entropy of a Linear layer over a large vocabulary without its [rows, V] logits in memory:
//   x = h W^T + b,  lse_r = log sum_v exp x_rv,  loss_r = lse_r - x_r,target,  loss = scale sum_r loss_r
//   D = softmax(x) - onehot(target) (zero rows where ignored),  dh = g D W,  dW = g D^T h,  db = g sum_r D,  g = grad_out scale
// Forward: one GEMM whose epilogue keeps, of every 64-column strip of a row, only its maximum and its sum of exponentials
// (8 bytes for 64 logits) and the target's logit; a second launch joins the strips.
// Backward: the vocabulary in pieces.  The logits of a piece are formed again, turned into D in the epilogue (16 bits), and multiplied
// while the cache still holds them; dh collects the pieces in fp32.  The bias gradient is summed from the unrounded D.  Every
// sum has a fixed order.
// All products are one GEMM kernel: C[m][n] = sum_k A[m][k] B[n][k] on the 16-bit matrix cores, fp32 accumulation.  An operand's k is
// contiguous (x), or its rows are k (W in dh, D and h in dW): those tiles pass the LDS's transposing read on their way to the matrix cores, and
// nothing is transposed in memory.
//   bf16: D is rounded to bf16 (2^-8 of each value, as much as the result's own rounding).
//   fp16: D 2^14 is rounded to fp16, so that a probability of 1e-8 still has full precision; the factor leaves again exactly.
//   fp32: every operand is the sum of two fp16 values (22 bits), scaled by a power of two so that its largest magnitude is near
//   2^14; the products hi hi + hi lo + lo hi drop 2^-22 of each term: as exact as an fp32 dot product, at three fp16
//   products for one (the fp32 matrix instruction takes sixteen times a 16-bit product).  For the logits every row of hidden and
//   every word of the weight has a scale of its own, so that no row touches another; as the contraction of dh and dW runs over words
//   and rows, those take one scale for all.  fp16 ends at 2^-24, so D 2^14 alone would hold 22 bits only of probabilities above 2^-17, and none
//   below 2^-39: the row of dW of a word that is no row's target (its probabilities may all be 1e-10) would be lost.  So each word's
//   column of D is multiplied by a power of two, its `lift`, that brings its largest value to 1; dW's row leaves it again in its epilogue, and for
//   dh the word's row of W is divided by it.  The largest probability of a word over all rows comes from a product of the high parts
//   alone, rounded up by what these may lack: 2^-10 of both rows' lengths (EP_TOP; 63 us at 4864 x 6756 x 512), where dW is wanted.  The values
//   may be up to 2^-17 below 1 then and still have their 22 bits.
// Rows that are left out are zeros in every operand that sums over rows, whatever they hold (NaN, infinities).
// Bound: the matrix cores (2 R E V flops a product; one forward, three backward of which the logits are repeated).
// Measured: 8192 rows x 65536 words x 2048, bf16: logits 1984 us (1108 TFLOP/s), a piece of 8192 words: D 266, dh 280, dW 257 (1033, 981, 1068);
// a library product reaches 1270.  4864 x 6756 x 512, fp32 as three fp16 products: logits 138 us (731), largest values 63,
// D 160, dh 132, dW 139.  684 x 81 x 512: 80 us in twelve launches.
#include "packed.hpp"

namespace icap {
namespace lce {

constexpr int BK = 64, ROWB = BK * 2;               // K tile; bytes of an LDS row
constexpr int STRIP = 64;                           // columns that share one (maximum, sum) pair
constexpr float D_SCALE = 16384.0f;                 // fp16 D
constexpr float LOG2E = 1.4426950408889634f;

enum Epilogue { EP_LSE, EP_GRAD, EP_OUT, EP_TOP };

struct Gemm {
    const unsigned short *a0, *a1, *b0, *b1;        // planes: high and (fp32 tensors) low parts
    long long lda, ldb;
    int M, N, K, pairs, ksplit, tiles_m, tiles_n;   // K % 64 == 0; pairs 1 or 3
    int a_cols, b_cols;                             // operands whose rows are k (K of them): columns there are (% 8 == 0)
    const float *urow, *ucol;                       // fp32: factors 2^-s of the logits' rows and columns
    // EP_LSE, EP_GRAD and EP_TOP
    const void* bias;                               // type of the tensors
    const long long* targets;
    long long ignore;
    int V, v0;                                      // column 0 of this product is word v0; words end at V
    float2* part; int strips; float* target_logit;  // EP_LSE
    const float* lse;                               // EP_GRAD, EP_TOP
    unsigned short *d0, *d1;                        // D [rows_pad][ldd], planes
    long long ldd;
    int rows_pad, cols_pad;                         // D is written (zeros) up to these multiples of 64
    float* colpart; long long ldc;                  // [row blocks][ldc]; EP_TOP: log2 of the largest magnitudes of D there
    const float* lift;                              // fp32: factors of D's columns (null: 1); EP_OUT: what the result's rows are divided by
    const float *nrow, *ncol;                       // EP_TOP: lengths of A's and B's rows, of which a product may lack their product times
    float lack;                                     // this
    // EP_OUT
    void* out; long long ldo;                       // final results (type of the tensors)
    float* acc; int accumulate;                     // or fp32 partial results [ksplit][M][N], added to what is there
    const float *f0, *f1, *f2;                      // final factor: product of these device scalars (null = 1) and f
    float f;
};

template <typename E> struct Mma;
template <> struct Mma<__bf16> {
    static __device__ __forceinline__ f32x16 go(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<_Float16> {
    static __device__ __forceinline__ f32x16 go(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ void load16(const void* g, unsigned char* lds_wave_base) {
    __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)(lds_wave_base), 16, 0, 0);
}

// accumulator row of register e, for lanes 0-31 (lanes 32-63: + 4)
__device__ __forceinline__ constexpr int acc_row(int e) { return (e & 3) + 8 * (e >> 2); }

// op over a lane and lane ^ 32
template <typename F>
__device__ __forceinline__ float other_half(float v, F op) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float final_factor(const Gemm& p) {
    float f = p.f;
    if (p.f0) f *= *p.f0;
    if (p.f1) f *= *p.f1;
    if (p.f2) f *= *p.f2;
    return f;
}

// op over the 32 lanes of a half
template <typename F>
__device__ __forceinline__ float half_wave(float v, F op) {
    v = op(v, dpp_f<DPP_QUAD_SWAP1>(v));
    v = op(v, dpp_f<DPP_QUAD_SWAP2>(v));
    v = op(v, dpp_f<DPP_HALF_MIRROR>(v));
    v = op(v, dpp_f<DPP_ROW_MIRROR>(v));
    return op(v, __shfl_xor(v, 16));
}

// high and low 16-bit parts of a value
template <typename E>
__device__ __forceinline__ void split(float x, E& hi, E& lo) {
    hi = (E)x;
    lo = (E)(x - (float)hi);
}

template <int BM, int BN, int ST> constexpr int smem_bytes() { return ST * (BM + BN) * ROWB; }

// WM x WN waves, each (BM / WM) x 64 of the tile.  Operands go global -> LDS without passing a register (16 bytes a lane, one wave
// 1 KB); ST - 1 K tiles are in flight while one multiplies; one wait and one barrier a K tile.  The 16-byte slot a lane
// fetches is permuted by its row, and the fragment reads apply the same permutation, so that 16 rows meet 16 different slots.
// AT, BT: the operand's rows are k.  Its tile is [64][BM]; a transposing read takes 64 bytes of four rows, which the permutation puts into
// different quarters of the LDS's 256-byte line.
template <int COLS> __device__ __forceinline__ int quarter(int k) { return COLS >= 128 ? (k & 3) << 2 : (k & 2) << 1; }

template <typename E, typename T, int BM, int BN, int WM, int WN, int ST, int EP, bool AT, bool BT>
__global__ __launch_bounds__(WM * WN * 64) void gemm_kernel(const Gemm p) {
    constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, RM = TM / 32, RN = 2, RPP = NW * 8;
    static_assert(TN == STRIP && TM % 32 == 0 && BM % RPP == 0 && BN % RPP == 0, "wave tiles");
    constexpr int APT = BM / RPP, BPT = BN / RPP, A_BYTES = BM * ROWB, STAGE = (BM + BN) * ROWB;
    constexpr int IMG = 9216, LD4 = TN + 4, LD2 = TN + 8;       // a wave's image of 32 rows: bytes; row lengths of fp32 and 16-bit ones
    static_assert(NW * IMG <= ST * STAGE && 32 * LD4 * 4 <= IMG && 2 * 32 * LD2 * 2 <= IMG, "the waves' result images fit the staging buffers");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave - wm * WN, lr = lane & 31, lh = lane >> 5;

    // each XCD (workgroups go round them) walks a contiguous range of tiles, four rows of tiles at a time: the 32 tiles of 256 x 256 that it
    // works on share 4 + 8 panels (with one column of all rows, 1 + 32, the last-level cache bound the long products: 4864 rows x 6756 words
    // of fp32 610 -> 587 us, 8192 x 65536 of bf16 8600 -> 8280)
    constexpr int GROUP = 4;
    const int nwg = gridDim.x, xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, tq = nwg >> 3, tr = nwg & 7;
    const int tlin = xcd * tq + (xcd < tr ? xcd : tr) + slot;
    const int group = tlin / (GROUP * p.tiles_n), in = tlin - group * (GROUP * p.tiles_n), gm = min(p.tiles_m - group * GROUP, GROUP);
    const int tile_n = in / gm, tile_m = group * GROUP + in - tile_n * gm;
    const int m0 = tile_m * BM, n0 = tile_n * BN;

    const int srow = wave * 8 + (lane >> 3), lslot = (lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7);
    // rows of k: a wave fetches 512 / BM of them at a time
    constexpr int ALR = BM / 8, BLR = BN / 8, AK = 64 / ALR, BKR = 64 / BLR;
    const int ak = wave * AK + lane / ALR, bk = wave * BKR + lane / BLR;        // + i NW AK: four rows' quarters are the same for every i
    static_assert(NW * AK % 4 == 0 && NW * BKR % 4 == 0, "permutation of the rows of k");
    const int acol = min(m0 + ((lane % ALR) ^ quarter<BM>(ak)) * 8, p.a_cols - 8), bcol = min(n0 + ((lane % BLR) ^ quarter<BN>(bk)) * 8, p.b_cols - 8);
    long long a_off[APT], b_off[BPT];
#pragma unroll
    for (int i = 0; i < APT; ++i) a_off[i] = AT ? (long long)(ak + i * NW * AK) * p.lda + acol : (long long)min(m0 + i * RPP + srow, p.M - 1) * p.lda + 8 * lslot;
#pragma unroll
    for (int i = 0; i < BPT; ++i) b_off[i] = BT ? (long long)(bk + i * NW * BKR) * p.ldb + bcol : (long long)min(n0 + i * RPP + srow, p.N - 1) * p.ldb + 8 * lslot;
    const int nk = p.K / BK, total = nk * p.pairs;
    const int per = (total + p.ksplit - 1) / p.ksplit, t_lo = min((int)blockIdx.y * per, total), t_hi = min(t_lo + per, total);
    int pair = t_lo / nk, kt = t_lo - pair * nk, left = t_hi - t_lo;
    auto issue = [&](int buf) __attribute__((always_inline)) {
        unsigned char* base = smem + buf * STAGE + wave * 1024;
        const unsigned short* a = (pair == 2 ? p.a1 : p.a0) + (AT ? kt * BK * p.lda : (long long)kt * BK);
        const unsigned short* b = (pair == 1 ? p.b1 : p.b0) + (BT ? kt * BK * p.ldb : (long long)kt * BK);
#pragma unroll
        for (int i = 0; i < APT; ++i) load16(a + a_off[i], base + i * (NW * 1024));
#pragma unroll
        for (int i = 0; i < BPT; ++i) load16(b + b_off[i], base + A_BYTES + i * (NW * 1024));
        if (--left > 0 && ++kt == nk) { kt = 0; ++pair; }       // behind the last tile it is fetched again, so that the waits can count
    };
    f32x16 acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int sw = (lr >> 1) & 7;
    // transposing reads: this lane's byte of a tile for the 32 columns from c, k 0 - 3 (+ 8 for lanes 32-63)
    const int tk = 8 * lh + ((lane & 15) >> 2), tslot = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    int at[RM], bt[RN];
#pragma unroll
    for (int i = 0; i < RM; ++i) at[i] = tk * BM * 2 + ((((wm * TM + i * 32) >> 3) + tslot) ^ quarter<BM>(tk)) * 16 + (lane & 1) * 8;
#pragma unroll
    for (int j = 0; j < RN; ++j) bt[j] = tk * BN * 2 + ((((wn * TN + j * 32) >> 3) + tslot) ^ quarter<BN>(tk)) * 16 + (lane & 1) * 8;
    auto turned = [&](const unsigned char* x, int row) __attribute__((always_inline)) {         // k 0 - 3 and 4 - 7 of one column
        typedef __attribute__((address_space(3))) i16x4* lds_ptr;
        typedef short i16x8 __attribute__((ext_vector_type(8)));
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)x), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(x + 4 * row));
        const i16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(typename Vec<E>::x8, both);
    };
    auto compute = [&](int buf) __attribute__((always_inline)) {
        const unsigned char* ta = smem + buf * STAGE;
        const unsigned char* tb = ta + A_BYTES;
        const unsigned char* sa = ta + (wm * TM + lr) * ROWB;
        const unsigned char* sb = tb + (wn * TN + lr) * ROWB;
#pragma unroll
        for (int s = 0; s < BK / 16; ++s) {
            const int off = ((2 * s + lh) ^ sw) * 16;
            typename Vec<E>::x8 af[RM], bf[RN];
#pragma unroll
            for (int i = 0; i < RM; ++i) {
                if constexpr (AT) af[i] = turned(ta + at[i] + s * 16 * BM * 2, BM * 2);
                else af[i] = *reinterpret_cast<const typename Vec<E>::x8*>(sa + i * 32 * ROWB + off);
            }
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                if constexpr (BT) bf[j] = turned(tb + bt[j] + s * 16 * BN * 2, BN * 2);
                else bf[j] = *reinterpret_cast<const typename Vec<E>::x8*>(sb + j * 32 * ROWB + off);
            }
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < RN; ++j) acc[i][j] = Mma<E>::go(bf[j], af[i], acc[i][j]);
        }
    };
    if (t_lo < t_hi) {
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) issue(i);
        int buf = 0;
        for (int t = t_lo; t < t_hi; ++t) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 2) * (APT + BPT)) : "memory");
            __builtin_amdgcn_s_barrier();       // K tile t is there for every wave, and everybody has left the buffer filled next
            asm volatile("" ::: "memory");
            issue(buf == 0 ? ST - 1 : buf - 1);
            compute(buf);
            buf = buf + 1 == ST ? 0 : buf + 1;
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // Epilogue, every wave on its own, 32 rows at a time.  The products were formed transposed (B's rows as the first operand), so a lane
    // holds row lane % 32 of C, columns 32 j + acc_row(e) + 4 (lane / 32): a row's statistics stay in two lanes, four
    // columns are neighbours, and what goes to memory passes the LDS in 8- and 16-byte pieces.
    unsigned char* img = smem + wave * IMG;
    const int nb = n0 + wn * TN;                                // the wave's first column
    const bool edge = nb + TN > p.N;                            // some columns do not exist
    // A column's 32 rows are spread over the 32 lanes of a half.  What they make of it is kept by one lane, the half's lr-th column by lane
    // lr, and stored at once (a store for each column: 89 us where this took 61, EP_TOP of 4864 x 6756 x 512)
    const int mine = nb + (lr >> 4) * 32 + ((lr >> 2) & 3) * 8 + 4 * lh + (lr & 3);
    if constexpr (EP == EP_TOP) {
        const float b = (p.bias && mine < p.N) ? (float)((const T*)p.bias)[p.v0 + mine] * LOG2E : 0.f;
        int t[RM];
        float ur[RM], nr[RM], lse2[RM], most = -INFINITY;
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            const int m = m0 + wm * TM + i * 32 + lr, mm = min(m, p.M - 1);
            const long long target = p.targets[mm];
            const bool on = m < p.M && target >= 0 && target < p.V && target != p.ignore;
            t[i] = on ? (int)target - p.v0 - nb - 4 * lh : -1;
            ur[i] = p.urow[mm] * LOG2E;
            nr[i] = p.nrow[mm] * p.lack * ur[i];
            lse2[i] = on ? p.lse[mm] * LOG2E : INFINITY;
        }
        f32x4 uc[RN][4], nc[RN][4];
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uc[j][g] = *reinterpret_cast<const f32x4*>(p.ucol + nb + j * 32 + 8 * g + 4 * lh);
                nc[j][g] = *reinterpret_cast<const f32x4*>(p.ncol + nb + j * 32 + 8 * g + 4 * lh) * uc[j][g];
            }
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                float v = -INFINITY;
#pragma unroll
                for (int i = 0; i < RM; ++i) {
                    const float l = fmaf(acc[i][j][k], uc[j][k >> 2][k & 3] * ur[i], fmaf(nc[j][k >> 2][k & 3], nr[i], -lse2[i]));
                    v = fmaxf(v, t[i] == j * 32 + acc_row(k) ? INFINITY : l);               // a target's |D| may be 1
                }
                v = half_wave(v, [](float a, float c) { return fmaxf(a, c); });
                most = lr == j * 16 + k ? v : most;
            }
        if (mine < p.N) p.colpart[(long long)(tile_m * WM + wm) * p.ldc + p.v0 + mine] = most + b;
    } else if constexpr (EP != EP_OUT) {
        f32x4 bias[RN][4];
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = nb + j * 32 + 8 * g + 4 * lh + e;
                    bias[j][g][e] = (p.bias && n < p.N) ? (float)((const T*)p.bias)[p.v0 + n] : 0.f;
                }
        f32x4 colsum[RN][4] = {};
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            const int mb = m0 + wm * TM + i * 32, m = mb + lr, mm = min(m, p.M - 1);
            const long long target = p.targets[mm];
            const int t = (target >= 0 && target < p.V) ? (int)target - p.v0 - nb : -1;         // the target's column of this strip
            float x[RN][16];
            if constexpr (sizeof(T) == 4) {
                const float ur = p.urow[mm];
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 f = *reinterpret_cast<const f32x4*>(p.ucol + nb + j * 32 + 8 * g + 4 * lh) * ur;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[j][4 * g + e] = fmaf(acc[i][j][4 * g + e], f[e], bias[j][g][e]);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[j][e] = acc[i][j][e] + bias[j][e >> 2][e & 3];
            }
            if (edge) {
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (j * 32 + acc_row(e) + 4 * lh >= p.N - nb) x[j][e] = -INFINITY;
            }
            if constexpr (EP == EP_LSE) {
                float mx = x[0][0];
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, x[j][e]);
                mx = other_half(mx, [](float a, float b) { return fmaxf(a, b); });
                const float base = mx == -INFINITY ? 0.f : mx * LOG2E;
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(fmaf(x[j][e], LOG2E, -base));
                s = other_half(s, [](float a, float b) { return a + b; });
                const int strip = tile_n * WN + wn;
                if (lh == 0 && m < p.M && strip < p.strips) p.part[(long long)m * p.strips + strip] = make_float2(mx, s);
                if (__any(t >= 0 && t < TN)) {
#pragma unroll
                    for (int j = 0; j < RN; ++j)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (t == j * 32 + acc_row(e) + 4 * lh && m < p.M) p.target_logit[m] = x[j][e];
                }
            } else {
                const bool on = m < p.M && target >= 0 && target < p.V && target != p.ignore;
                const float lse2 = p.lse[mm] * LOG2E;
                const bool here = __any(t >= 0 && t < TN);
                E* hi = reinterpret_cast<E*>(img);
                E* lo = hi + 32 * LD2;
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        typename Vec<E>::x4 h4, l4;
                        f32x4 up = {D_SCALE, D_SCALE, D_SCALE, D_SCALE};
                        if constexpr (sizeof(T) == 4)
                            if (p.lift) up *= *reinterpret_cast<const f32x4*>(p.lift + nb + j * 32 + 8 * g + 4 * lh);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float d = __builtin_amdgcn_exp2f(fmaf(x[j][4 * g + e], LOG2E, -lse2));
                            if (here && t == j * 32 + 8 * g + 4 * lh + e) d -= 1.0f;
                            d = on ? d : 0.f;
                            colsum[j][g][e] += d;
                            if constexpr (!__is_same(E, __bf16)) d *= up[e];
                            E h, l;
                            split<E>(d, h, l);
                            h4[e] = h;
                            l4[e] = l;
                        }
                        *reinterpret_cast<typename Vec<E>::x4*>(hi + lr * LD2 + j * 32 + 8 * g + 4 * lh) = h4;
                        if constexpr (sizeof(T) == 4) *reinterpret_cast<typename Vec<E>::x4*>(lo + lr * LD2 + j * 32 + 8 * g + 4 * lh) = l4;
                    }
#pragma unroll
                for (int part = 0; part < (sizeof(T) == 4 ? 2 : 1); ++part) {
                    const E* im = part ? lo : hi;
                    unsigned short* d = part ? p.d1 : p.d0;
                    // rows: eight lanes of 16 bytes each
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int row = q * 8 + (lane >> 3), c = (lane & 7) * 8;
                        if (mb + row < p.rows_pad && nb + c < p.cols_pad)
                            *reinterpret_cast<u32x4*>(d + (long long)(mb + row) * p.ldd + nb + c) = *reinterpret_cast<const u32x4*>(im + row * LD2 + c);
                    }
                }
            }
        }
        if constexpr (EP == EP_GRAD) {
            if (p.colpart) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float v = half_wave(colsum[j][k >> 2][k & 3], [](float a, float c) { return a + c; });
                        sum = lr == j * 16 + k ? v : sum;
                    }
                if (mine < p.N) p.colpart[(long long)(tile_m * WM + wm) * p.ldc + p.v0 + mine] = sum;
            }
        }
    } else {
        const float f = p.acc ? 1.0f : final_factor(p);
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            const int mb = m0 + wm * TM + i * 32;
            if (sizeof(T) == 4 || p.acc) {
                float* im = reinterpret_cast<float*>(img);
                float fr = f;
                if constexpr (sizeof(T) == 4)
                    if (p.lift) fr = f / p.lift[min(mb + lr, p.M - 1)];         // powers of two
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<f32x4*>(im + lr * LD4 + j * 32 + 8 * g + 4 * lh) =
                            f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]} * fr;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const int row = q * 4 + (lane >> 4), c = (lane & 15) * 4, m = mb + row, n = nb + c;
                    f32x4 v = *reinterpret_cast<const f32x4*>(im + row * LD4 + c);
                    if (m >= p.M || n >= p.N) continue;
                    float* o = p.acc ? p.acc + ((long long)blockIdx.y * p.M + m) * p.N + n : (float*)p.out + (long long)m * p.ldo + n;
                    const bool add = p.acc && p.accumulate;
                    if (p.N % 4 == 0) {
                        if (add) v += *reinterpret_cast<const f32x4*>(o);
                        *reinterpret_cast<f32x4*>(o) = v;
                    } else {
                        for (int e = 0; e < 4 && n + e < p.N; ++e) o[e] = add ? o[e] + v[e] : v[e];
                    }
                }
            } else if constexpr (sizeof(T) == 2) {
                T* im = reinterpret_cast<T*>(img);
#pragma unroll
                for (int j = 0; j < RN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<typename Vec<T>::x4*>(im + lr * LD2 + j * 32 + 8 * g + 4 * lh) =
                            __builtin_convertvector(f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]} * f, typename Vec<T>::x4);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = q * 8 + (lane >> 3), c = (lane & 7) * 8, m = mb + row, n = nb + c;
                    const typename Vec<T>::x8 v = *reinterpret_cast<const typename Vec<T>::x8*>(im + row * LD2 + c);
                    if (m >= p.M || n >= p.N) continue;
                    T* o = (T*)p.out + (long long)m * p.ldo + n;
                    if (p.N % 8 == 0) *reinterpret_cast<typename Vec<T>::x8*>(o) = v;
                    else
                        for (int e = 0; e < 8 && n + e < p.N; ++e) o[e] = v[e];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ joining the strips
// one wave a row: lse and loss of the row
__global__ __launch_bounds__(256) void lse_kernel(const float2* part, int strips, const float* target_logit, const long long* targets, int R,
                                                  int V, long long ignore, float* row_loss, float* row_lse) {
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= R) return;
    const float2* p = part + (long long)r * strips;
    float m = -INFINITY;
    for (int i = lane; i < strips; i += 64) m = fmaxf(m, p[i].x);
    m = wave_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    for (int i = lane; i < strips; i += 64) s += p[i].y * __builtin_amdgcn_exp2f((p[i].x - base) * LOG2E);
    s = wave_sum(s);
    if (lane == 0) {
        const float lse = m + logf(s);
        const long long t = targets[r];
        row_lse[r] = lse;
        row_loss[r] = (t >= 0 && t < V && t != ignore) ? lse - target_logit[r] : 0.f;
    }
}

// largest of n values >= 0, by 1024 threads
__device__ __forceinline__ float block_max(const float* x, int n, float* red) {
    float m = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 1024) m = fmaxf(m, x[i]);
    m = wave_max(m);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int i = 0; i < 16; ++i) m = fmaxf(m, red[i]);
    return m;
}

// loss (its sum in 64 bits) and the scale of every row; fp32 (urow, ucol): the scales of whole tensors, from those of their rows
__global__ __launch_bounds__(1024) void loss_kernel(const float* row_loss, const long long* targets, int R, int V, long long ignore, int mean_over_valid,
                                                    const float* urow, const float* ucol, float* loss, float* out) {
    __shared__ double ss[16];
    __shared__ int sc[16];
    if (urow) {
        __shared__ float red[16];
        const float h = block_max(urow, R, red), w = block_max(ucol, V, red);
        if (threadIdx.x == 0) { out[2] = 1.0f / h; out[3] = h; out[4] = 1.0f / w; out[5] = w; }
    }
    double s = 0.0;
    int c = 0;
#pragma unroll 8
    for (int r = threadIdx.x; r < R; r += 1024) {
        s += row_loss[r];
        const long long t = targets[r];
        c += (t >= 0 && t < V && t != ignore) ? 1 : 0;
    }
    for (int d = 32; d; d >>= 1) { s += __shfl_xor(s, d); c += __shfl_xor(c, d); }
    if ((threadIdx.x & 63) == 0) { ss[threadIdx.x >> 6] = s; sc[threadIdx.x >> 6] = c; }
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        int cnt = 0;
        for (int i = 0; i < 16; ++i) { sum += ss[i]; cnt += sc[i]; }
        const int over = mean_over_valid ? cnt : R;
        out[0] = over > 0 ? (float)(sum / over) : 0.f;
        if (loss) *loss = out[0];
        out[1] = over > 0 ? 1.0f / (float)over : 0.f;
    }
}

// ------------------------------------------------------------------------------------------------ operands
// 2^-s for values whose largest magnitude is m: 2^s brings it to [2^13, 2^14].  Within 2^+-60, so that factors and their product stay
// fp32 values; nothing but zeros: the smallest factor, which no other row's exceeds.
__device__ __forceinline__ float unscale_of(float m) {
    if (!(m < INFINITY)) return 1.0f;                       // the row's result is not finite, whatever the scale
    return m > 0.f ? ldexpf(1.0f, min(max(ilogbf(m) + 1, -46), 74) - 14) : ldexpf(1.0f, -60);
}

// One matrix [R][C] (rows ld apart) and the 16-bit planes wanted of it, [.][Cp] with zeros from C on: r0, r1 for x (fp32: u the rows' factors
// 2^-s, found by the forward call), c0, c1 for the products that sum over rows (fp32: scale the whole tensor's 2^s), with zeros in rows R to
// Rp.  targets: rows left out are zeros.  Planes that are null are not wanted.  top (fp32): log2 of the largest magnitude of a word's column of
// D in each block of rows, of which the word's lift is made; its row of c0, c1 is divided by it.
struct Planes {
    const void* src; long long ld; int R, C, Rp, Cp;
    float* u; const float* scale;
    const long long* targets; int words; long long ignore;
    void *r0, *r1, *c0, *c1;
    const float* top; int blocks;
    float *lift, *norm;                             // norm: wanted lengths of r0, r1's rows
};

// the rows of both matrices, one wave a row; FIND: the rows' factors are found first
template <typename T, typename E, bool FIND>
__global__ __launch_bounds__(256) void planes_kernel(const Planes a, const Planes b) {
    constexpr int V = 16 / sizeof(T);                   // values of a 16-byte load
    const int lane = threadIdx.x & 63;
    int r = blockIdx.x * 4 + (threadIdx.x >> 6);
    const bool second = r >= a.Rp;
    const Planes& p = second ? b : a;
    if (second) r -= a.Rp;
    if (r >= p.Rp) return;
    const T* src = (const T*)p.src + (long long)r * p.ld;
    bool in = r < p.R;
    if (in && p.targets) {
        const long long t = p.targets[r];
        in = t >= 0 && t < p.words && t != p.ignore;
    }
    const bool vec = p.ld % V == 0 && p.C % V == 0 && (reinterpret_cast<uintptr_t>(p.src) & 15) == 0;
    auto at = [&](int c, T (&x)[V]) __attribute__((always_inline)) {
        if (vec && in && c < p.C) *reinterpret_cast<u32x4*>(x) = *reinterpret_cast<const u32x4*>(src + c);
        else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = (in && c + e < p.C) ? src[c + e] : (T)0.f;
        }
    };
    float u = 1.0f;
    if constexpr (FIND) {
        float m = 0.f;
#pragma unroll 4
        for (int c = lane * V; c < p.C; c += 64 * V) {
            T x[V];
            at(c, x);
#pragma unroll
            for (int e = 0; e < V; ++e) m = fmaxf(m, fabsf(x[e]));
        }
        u = unscale_of(wave_max(m));
        if (lane == 0 && r < p.R) p.u[r] = u;
    } else if (sizeof(T) == 4 && p.u && r < p.R) u = p.u[r];
    float f[2] = {1.0f / u, p.scale ? *p.scale : 1.0f};
    if (sizeof(T) == 4 && !FIND && p.lift) {
        float m = -INFINITY;
        if (r < p.R)
            for (int b = lane; b < p.blocks; b += 64) m = fmaxf(m, p.top[(long long)b * p.R + r]);
        m = wave_max(m);
        // to at most 1; not beyond 2^100, so that its inverse stays a factor; a column of zeros (and words that do not exist): 1
        const float lift = (m < 0.f && m > -INFINITY) ? ldexpf(1.0f, (int)fminf(-ceilf(m), 100.0f)) : 1.0f;
        if (lane == 0) p.lift[r] = lift;
        f[1] /= lift;
    }
    float squares = 0.f;
#pragma unroll 4
    for (int c = lane * V; c < p.Cp; c += 64 * V) {
        const long long to = (long long)r * p.Cp + c;
        T x[V];
        at(c, x);
        if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x4*>((E*)p.r0 + to) = *reinterpret_cast<u32x4*>(x);
        else {
            E h[V], l[V];
#pragma unroll
            for (int k = 0; k < (FIND ? 1 : 2); ++k) {
                if (k == 0 ? r >= p.R || !p.r0 : !p.c0) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float y = x[e] * f[k];
                    split<E>(y, h[e], l[e]);
                    if (!FIND && k == 0) squares = fmaf(y, y, squares);
                }
                *reinterpret_cast<u32x2*>((E*)(k ? p.c0 : p.r0) + to) = *reinterpret_cast<u32x2*>(h);
                *reinterpret_cast<u32x2*>((E*)(k ? p.c1 : p.r1) + to) = *reinterpret_cast<u32x2*>(l);
            }
        }
    }
    if (sizeof(T) == 4 && !FIND && p.norm) {
        squares = wave_sum(squares);
        if (lane == 0 && r < p.R) p.norm[r] = sqrtf(squares);
    }
}

// out[i] = factor * sum over splits of acc[split][i], in order; V values a thread (n % V == 0)
template <typename T, int V>
__global__ __launch_bounds__(256) void join_kernel(const float* acc, int splits, long long n, T* out, const Gemm p) {
    typedef float vec __attribute__((ext_vector_type(V)));
    typedef T tvec __attribute__((ext_vector_type(V)));
    const float f = final_factor(p);
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * V; i < n; i += (long long)gridDim.x * 256 * V) {
        vec s = *reinterpret_cast<const vec*>(acc + i);
#pragma unroll 8
        for (int z = 1; z < splits; ++z) s += *reinterpret_cast<const vec*>(acc + z * n + i);
        *reinterpret_cast<tvec*>(out + i) = __builtin_convertvector(s * f, tvec);
    }
}

// 64 columns a workgroup, four parts of the row blocks each
template <typename T>
__global__ __launch_bounds__(256) void bias_kernel(const float* colpart, int blocks, int V, T* out, const float* f0, const float* f1) {
    __shared__ float part[4][64];
    const int c = threadIdx.x & 63, v = blockIdx.x * 64 + c, q = threadIdx.x >> 6, per = (blocks + 3) / 4;
    float s = 0.f;
    if (v < V) {
#pragma unroll 16
        for (int b = q * per; b < min(q * per + per, blocks); ++b) s += colpart[(long long)b * V + v];
    }
    part[q][c] = s;
    __syncthreads();
    if (q == 0 && v < V) out[v] = (T)((((part[0][c] + part[1][c]) + part[2][c]) + part[3][c]) * (*f0 * *f1));
}

// ------------------------------------------------------------------------------------------------ host
inline long long up(long long x, long long m) { return (x + m - 1) / m * m; }

// workspace: parts one after another, each on a 256-byte border; with base null only their sizes are counted
struct Space {
    char* base;
    long long at = 0;
    template <typename X> X* take(long long n) {
        X* p = base ? reinterpret_cast<X*>(base + at) : nullptr;
        at += up(n * (long long)sizeof(X), 256);
        return p;
    }
};

// Tile of a GEMM and the pieces of its contraction.  Measured on whole cards of tiles (us a K tile of 64 of every tile that runs at once) and
// on a few of them alone: 256 x 256 with eight waves, one workgroup a CU: 1.9 / 1.6; 128 x 128 with four, two a CU: 1.2 / 0.7; 64 x 64
// with two, two a CU, three K tiles in flight: 0.65 / 0.4 (at 8192 x 2048 x 8192: 1140, 890 and 440 TFLOP/s).  A round of tiles begins
// and ends with some 4 us.  Pieces of the contraction cost a pass over their fp32 results.  The cheapest of these sums is taken.
struct Shape { int tile, tiles_m, tiles_n, splits; };
inline Shape resized(const Shape& s, int M, int N) { return {s.tile, (int)(up(M, s.tile) / s.tile), (int)(up(N, s.tile) / s.tile), s.splits}; }
inline Shape shape_of(long long M, long long N, long long ktiles, bool may_split) {
    static const struct { int tile, slots; double full, few; } cfg[3] = {{256, 256, 1.9, 1.6}, {128, 512, 1.2, 0.7}, {64, 512, 0.65, 0.4}};
    Shape best{};
    double least = 0.0;
    for (const auto& c : cfg) {
        const long long tiles = up(M, c.tile) / c.tile * (up(N, c.tile) / c.tile);
        for (int k = 1; k <= (may_split ? 32 : 1) && (k == 1 || ktiles / k >= 4); ++k) {
            const long long wgs = tiles * k, rounds = (wgs + c.slots - 1) / c.slots;
            const double fill = rounds > 1 ? 1.0 : (double)wgs / c.slots, each = c.few + (c.full - c.few) * fill;
            const double cost = rounds * (4.0 + (double)((ktiles + k - 1) / k) * each) + (k > 1 ? 4.0 + (double)M * N * 4.0 * (k + 1) / 3e6 : 0.0);
            if (best.tile == 0 || cost < least) {
                least = cost;
                best = {c.tile, (int)(up(M, c.tile) / c.tile), (int)(up(N, c.tile) / c.tile), k};
            }
        }
    }
    return best;
}

template <typename E, typename T, int BM, int BN, int WM, int WN, int ST, int EP, bool AT, bool BT>
int go(const Gemm& p, hipStream_t st) {
    static const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_kernel<E, T, BM, BN, WM, WN, ST, EP, AT, BT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<BM, BN, ST>());
    if (rc != hipSuccess) { set_error("linear_ce: cannot raise the dynamic LDS limit: %s", hipGetErrorString(rc)); return ICAP_ERR_HIP_BASE + (int)rc; }
    hipLaunchKernelGGL((gemm_kernel<E, T, BM, BN, WM, WN, ST, EP, AT, BT>), dim3((unsigned)(p.tiles_m * p.tiles_n), p.ksplit), dim3(WM * WN * 64),
                       (smem_bytes<BM, BN, ST>()), st, p);
    return launch_status("linear_ce");
}

template <typename E, typename T, int EP, bool AT = false, bool BT = false>
int gemm(Gemm& p, const Shape& s, hipStream_t st) {
    p.tiles_m = s.tiles_m;
    p.tiles_n = s.tiles_n;
    p.ksplit = s.splits;
    if (s.tile == 256) return go<E, T, 256, 256, 2, 4, 2, EP, AT, BT>(p, st);
    if (s.tile == 128) return go<E, T, 128, 128, 2, 2, 2, EP, AT, BT>(p, st);
    return go<E, T, 64, 64, 2, 1, 4, EP, AT, BT>(p, st);
}

struct Call {
    const void *h, *w, *bias;
    long long ld_h, ld_w;
    const long long* targets;
    int R, E, V;
    long long ignore;
    int need = 0;                       // the backward call's results that are wanted; 0: the forward call
};
enum { NEED_DH = 1, NEED_DW = 2, NEED_DB = 4 };

// Bytes of D that a piece of the vocabulary may take.  The last-level cache holds 256 MB: up to there in one piece (131 MB at 4864 rows x 6756
// words: 609 us, in two pieces 676), otherwise in pieces of half of it, beside which the operands stay (8192 x 65536, 1 GB: 8436 us,
// with pieces of 256 MB 8740, of 512 MB 8700).
constexpr long long WHOLE_BYTES = 256ll << 20, PIECE_BYTES = 128ll << 20;

template <typename T> struct Of { typedef T E; static constexpr int planes = 1; };
template <> struct Of<float> { typedef _Float16 E; static constexpr int planes = 2; };

// whether a matrix can be read by the GEMM as it is: 16 bits, rows of whole 64-value K tiles, 16-byte pieces
template <typename T>
bool direct(const void* x, long long ld, int C) { return sizeof(T) == 2 && C % 64 == 0 && ld % 8 == 0 && aligned16(x); }

// the 16-bit planes of a matrix: row0, row1 for x; sum0, sum1 for the products that sum over its rows
template <typename T>
struct Operand {
    typename Of<T>::E *row0 = nullptr, *row1 = nullptr, *sum0 = nullptr, *sum1 = nullptr;
    long long ld = 0;
};

// room for them; Rp: rows with those that are zeros; sums: those planes are wanted
template <typename T>
Operand<T> room(Space& ws, const void* x, long long ld, int Rp, int C, bool sums, bool is_direct) {
    typedef typename Of<T>::E E;
    Operand<T> o;
    o.ld = up(C, 64);
    if (is_direct) { o.row0 = (E*)const_cast<void*>(x); o.ld = ld; }
    else o.row0 = ws.take<E>(Rp * o.ld);
    if (Of<T>::planes == 2) o.row1 = ws.take<E>(Rp * o.ld);
    o.sum0 = o.row0;
    if (Of<T>::planes == 2) o.sum0 = nullptr;
    if (Of<T>::planes == 2 && sums) { o.sum0 = ws.take<E>(Rp * o.ld); o.sum1 = ws.take<E>(Rp * o.ld); }
    return o;
}

template <typename T>
Planes planes_of(const Operand<T>& o, const void* x, long long ld, int R, int Rp, int C, bool is_direct, float* u, const float* scale) {
    return {x, ld, R, C, is_direct ? 0 : Rp, (int)up(C, 64), u, scale, nullptr, 0, 0, o.row0, o.row1, o.sum0, o.sum1, nullptr, 0, nullptr, nullptr};
}

template <typename T>
struct Plan {
    bool h_direct, w_direct;
    Operand<T> h, w;
    // forward
    float2* part; float* target_logit; int strips;
    // backward
    int piece; long long ldd;
    typename Of<T>::E *d0, *d1;
    float *colpart, *acc_h, *acc_w, *lift, *norm_h, *norm_w;
    Shape s_top, s_logit, s_h, s_w;
    long long bytes;

    // any: whatever the addresses and row distances
    Plan(const Call& c, char* base, bool any = false) {
        typedef typename Of<T>::E E;
        const bool backward = c.need != 0, dh = c.need & NEED_DH, dw = c.need & NEED_DW;
        Space ws{base};
        h_direct = !backward && direct<T>(c.h, c.ld_h, c.E);        // dW needs zeros in the rows that are left out
        w_direct = direct<T>(c.w, c.ld_w, c.E) && (!backward || c.V % 64 == 0);          // dh reads whole K tiles of words
        if (any) h_direct = w_direct = false;
        h = room<T>(ws, c.h, c.ld_h, backward ? (int)up(c.R, 64) : c.R, c.E, dw, h_direct);
        w = room<T>(ws, c.w, c.ld_w, backward ? (int)up(c.V, 64) : c.V, c.E, dh, w_direct);
        const int pairs = Of<T>::planes == 2 ? 3 : 1;
        if (!backward) {
            s_logit = shape_of(c.R, c.V, up(c.E, 64) / 64 * pairs, false);
            strips = (int)(up(c.V, STRIP) / STRIP);
            part = ws.take<float2>((long long)c.R * strips);
            target_logit = ws.take<float>(c.R);
        } else {
            const long long rp = up(c.R, 64);
            const long long word = rp * 2 * Of<T>::planes;
            long long v = (word * c.V <= WHOLE_BYTES ? WHOLE_BYTES : PIECE_BYTES) / word / 256 * 256;
            if (v < 256) v = 256;
            if (v >= c.V) v = c.V;
            else v = up((c.V + (c.V + v - 1) / v - 1) / ((c.V + v - 1) / v), 256);      // pieces of about the same size
            piece = (int)v;
            ldd = up(piece, 64);
            d0 = ws.take<E>(rp * ldd);
            d1 = Of<T>::planes == 2 ? ws.take<E>(rp * ldd) : nullptr;
            s_logit = shape_of(c.R, piece, up(c.E, 64) / 64 * pairs, false);
            s_h = shape_of(c.R, c.E, ldd / 64 * pairs, true);
            s_w = shape_of(piece, c.E, rp / 64 * pairs, true);
            // the largest values of D's columns, once they have become factors, make room for the columns' sums
            int blocks = c.need & NEED_DB ? s_logit.tiles_m * 2 : 0;
            lift = norm_h = norm_w = nullptr;
            if (Of<T>::planes == 2 && dw) {
                s_top = shape_of(c.R, c.V, up(c.E, 64) / 64, false);
                if (s_top.tiles_m * 2 > blocks) blocks = s_top.tiles_m * 2;
                lift = ws.take<float>(up(c.V, 64) + 256);       // these are read up to 256 behind the last, too
                norm_h = ws.take<float>(up(c.R, 64));
                norm_w = ws.take<float>(up(c.V, 64) + 256);
            }
            colpart = ws.take<float>((long long)blocks * c.V);
            acc_h = ws.take<float>(dh && (s_h.splits > 1 || piece < c.V) ? (long long)s_h.splits * c.R * c.E : 0);
            acc_w = ws.take<float>(dw && s_w.splits > 1 ? (long long)s_w.splits * piece * c.E : 0);
        }
        bytes = ws.at;
    }
};

// The forward call's results: loss, scale of a row, and of fp32 tensors (for the backward call) the tensors' scales 2^s_h, 2^-s_h, 2^s_w,
// 2^-s_w, and from OUT_ROWS on the factors 2^-s of every row of hidden, then of every word (read up to 256 behind the last)
constexpr int OUT_ROWS = 8;
inline long long out_floats(int dtype, int R, int V) { return OUT_ROWS + (dtype == DT_F32 ? up(R, 64) + up(V, 64) + 256 : 0); }

// lifted: the sums' planes of the weight come later (words)
template <typename T>
void operands(const Call& c, Plan<T>& p, float* out, bool backward, bool lifted, hipStream_t st) {
    float *uh = nullptr, *uw = nullptr;
    if constexpr (sizeof(T) == 4) { uh = out + OUT_ROWS; uw = uh + up(c.R, 64); }
    Planes a = planes_of<T>(p.h, c.h, c.ld_h, c.R, backward ? (int)up(c.R, 64) : c.R, c.E, p.h_direct, uh, uh && backward ? out + 2 : nullptr);
    Planes b = planes_of<T>(p.w, c.w, c.ld_w, c.V, backward ? (int)up(c.V, 64) : c.V, c.E, p.w_direct, uw, uw && backward ? out + 4 : nullptr);
    if (lifted) { b.Rp = c.V; b.c0 = b.c1 = nullptr; a.norm = p.norm_h; b.norm = p.norm_w; }
    a.targets = c.targets;
    a.words = c.V;
    a.ignore = c.ignore;
    const long long rows = (long long)a.Rp + b.Rp;
    if (rows == 0) return;
    const dim3 grid((unsigned)((rows + 3) / 4));
    if (sizeof(T) == 4 && !backward) hipLaunchKernelGGL((planes_kernel<T, typename Of<T>::E, sizeof(T) == 4>), grid, dim3(256), 0, st, a, b);
    else hipLaunchKernelGGL((planes_kernel<T, typename Of<T>::E, false>), grid, dim3(256), 0, st, a, b);
}

// fp32: the words' lifts, from what EP_TOP found, and with them (dh wanted) the planes of the weight for dh
template <typename T>
void words(const Call& c, Plan<T>& p, const float* meta, bool dh, hipStream_t st) {
    Planes a = planes_of<T>(p.w, c.w, c.ld_w, c.V, (int)up(c.V, 64), c.E, false, nullptr, meta + 4), none{};
    a.r0 = a.r1 = nullptr;
    if (!dh) { a.c0 = a.c1 = nullptr; a.Cp = 0; }
    a.top = p.colpart;
    a.blocks = p.s_top.tiles_m * 2;
    a.lift = p.lift;
    hipLaunchKernelGGL((planes_kernel<T, typename Of<T>::E, false>), dim3((unsigned)((a.Rp + 3) / 4)), dim3(256), 0, st, a, none);
}

template <typename T>
Gemm logits(const Call& c, const Plan<T>& p, const float* out, int v0, int vn) {
    Gemm g{};
    g.a0 = (const unsigned short*)p.h.row0;
    g.a1 = (const unsigned short*)p.h.row1;
    g.b0 = (const unsigned short*)p.w.row0 + v0 * p.w.ld;
    g.b1 = p.w.row1 ? (const unsigned short*)p.w.row1 + v0 * p.w.ld : nullptr;
    g.lda = p.h.ld;
    g.ldb = p.w.ld;
    g.M = c.R; g.N = vn; g.K = (int)up(c.E, 64);
    g.pairs = Of<T>::planes == 2 ? 3 : 1;
    if (sizeof(T) == 4) { g.urow = out + OUT_ROWS; g.ucol = g.urow + up(c.R, 64) + v0; }
    g.bias = c.bias; g.targets = c.targets; g.ignore = c.ignore; g.V = c.V; g.v0 = v0;
    return g;
}

template <typename T>
int fwd(const Call& c, int mean_over_valid, float* row_loss, float* row_lse, float* loss, float* out, char* ws, hipStream_t st) {
    typedef typename Of<T>::E E;
    Plan<T> p(c, ws);
    operands<T>(c, p, out, false, false, st);
    Gemm g = logits<T>(c, p, out, 0, c.V);
    g.part = p.part; g.strips = p.strips; g.target_logit = p.target_logit;
    if (int rc = gemm<E, T, EP_LSE>(g, p.s_logit, st)) return rc;
    hipLaunchKernelGGL(lse_kernel, dim3((c.R + 3) / 4), dim3(256), 0, st, p.part, p.strips, p.target_logit, c.targets, c.R, c.V, c.ignore, row_loss, row_lse);
    hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, row_loss, c.targets, c.R, c.V, c.ignore, mean_over_valid, g.urow, g.ucol, loss, out);
    return launch_status("linear_ce_fwd");
}

template <typename T>
void join(const float* acc, int splits, long long n, T* out, const Gemm& p, hipStream_t st) {
    const long long blocks = up(n, n % 4 == 0 ? 1024 : 256) / (n % 4 == 0 ? 1024 : 256);
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
    if (n % 4 == 0) hipLaunchKernelGGL((join_kernel<T, 4>), grid, dim3(256), 0, st, acc, splits, n, out, p);
    else hipLaunchKernelGGL((join_kernel<T, 1>), grid, dim3(256), 0, st, acc, splits, n, out, p);
}

template <typename T>
int bwd(const Call& c, const float* row_lse, const float* meta, const float* grad_out, void* dh, void* dw, void* db, char* ws, hipStream_t st) {
    typedef typename Of<T>::E E;
    Plan<T> p(c, ws);
    const bool lifted = sizeof(T) == 4 && dw;
    operands<T>(c, p, const_cast<float*>(meta), true, lifted, st);         // which only reads it here
    if constexpr (sizeof(T) == 4)
        if (lifted) {
            Gemm g = logits<T>(c, p, meta, 0, c.V);
            g.lse = row_lse;
            g.pairs = 1;
            g.nrow = p.norm_h; g.ncol = p.norm_w;
            g.lack = 0x1.04p-10f + (float)c.E * 0x1p-24f;           // both sides' low parts, and the sum's own roundings
            g.colpart = p.colpart; g.ldc = c.V;
            if (int rc = gemm<E, T, EP_TOP>(g, p.s_top, st)) return rc;
            words<T>(c, p, meta, dh, st);
        }
    const float back = __is_same(E, _Float16) ? 1.0f / D_SCALE : 1.0f;
    for (int v0 = 0; v0 < c.V; v0 += p.piece) {
        const int vn = c.V - v0 < p.piece ? c.V - v0 : p.piece;
        Gemm g = logits<T>(c, p, meta, v0, vn);
        g.lse = row_lse;
        g.d0 = (unsigned short*)p.d0; g.d1 = (unsigned short*)p.d1;
        g.ldd = p.ldd;
        g.rows_pad = (int)up(c.R, 64); g.cols_pad = (int)up(vn, 64);
        g.colpart = db ? p.colpart : nullptr; g.ldc = c.V;
        g.lift = lifted ? p.lift + v0 : nullptr;
        if (int rc = gemm<E, T, EP_GRAD>(g, resized(p.s_logit, c.R, vn), st)) return rc;
        if (dh) {
            Gemm q{};
            q.a0 = (const unsigned short*)p.d0; q.a1 = (const unsigned short*)p.d1;
            q.b0 = (const unsigned short*)p.w.sum0 + v0 * p.w.ld; q.b1 = p.w.sum1 ? (const unsigned short*)p.w.sum1 + v0 * p.w.ld : nullptr;
            q.lda = p.ldd; q.ldb = p.w.ld;
            q.M = c.R; q.N = c.E; q.K = (int)up(vn, 64);
            q.b_cols = (int)up(c.E, 64);
            q.pairs = g.pairs;
            q.f0 = grad_out; q.f1 = meta + 1; q.f2 = sizeof(T) == 4 ? meta + 5 : nullptr; q.f = back;
            const bool whole = p.s_h.splits == 1 && p.piece >= c.V;
            if (whole) { q.out = dh; q.ldo = c.E; }
            else { q.acc = p.acc_h; q.accumulate = v0 > 0; }
            if (int rc = gemm<E, T, EP_OUT, false, true>(q, p.s_h, st)) return rc;
            if (!whole && v0 + vn == c.V) {
                join(p.acc_h, p.s_h.splits, (long long)c.R * c.E, (T*)dh, q, st);
            }
        }
        if (dw) {
            Gemm q{};
            q.a0 = (const unsigned short*)p.d0; q.a1 = (const unsigned short*)p.d1;
            q.b0 = (const unsigned short*)p.h.sum0; q.b1 = (const unsigned short*)p.h.sum1;
            q.lda = p.ldd; q.ldb = p.h.ld;
            q.M = vn; q.N = c.E; q.K = (int)up(c.R, 64);
            q.a_cols = (int)up(vn, 64); q.b_cols = (int)up(c.E, 64);
            q.pairs = g.pairs;
            q.f0 = grad_out; q.f1 = meta + 1; q.f2 = sizeof(T) == 4 ? meta + 3 : nullptr; q.f = back;
            q.lift = g.lift;
            T* dst = (T*)dw + (long long)v0 * c.E;
            if (p.s_w.splits == 1) { q.out = dst; q.ldo = c.E; }
            else q.acc = p.acc_w;
            if (int rc = gemm<E, T, EP_OUT, true, true>(q, resized(p.s_w, vn, c.E), st)) return rc;
            if (p.s_w.splits > 1) {
                join(p.acc_w, p.s_w.splits, (long long)vn * c.E, dst, q, st);
            }
        }
    }
    if (db)
        hipLaunchKernelGGL((bias_kernel<T>), dim3((c.V + 63) / 64), dim3(256), 0, st, p.colpart, p.s_logit.tiles_m * 2, c.V, (T*)db, grad_out, meta + 1);
    return launch_status("linear_ce_bwd");
}

static int check(int dtype, const Call& c, const char* what) {
    if (dtype < 0 || dtype > 2) { set_error("%s: unknown type %d", what, dtype); return ICAP_ERR_ARG; }
    if (!c.h || !c.w || !c.targets || c.R <= 0 || c.E <= 0 || c.V <= 0 || c.ld_h < c.E || c.ld_w < c.E) {
        set_error("%s: null tensor, empty size or overlapping rows", what);
        return ICAP_ERR_ARG;
    }
    // a launch has fewer than 2^32 threads
    const auto fits = [&](long long m, long long n, long long k) {
        const Shape t = shape_of(m, n, up(k, 64) / 64, false);
        return (long long)t.tiles_m * t.tiles_n * (t.tile == 64 ? 128 : t.tile == 128 ? 256 : 512) < (1ll << 32);
    };
    if (c.R > 65535 * 64 || c.E > (1 << 20) || c.V > 65535 * 64 || !fits(c.R, c.V, dtype == DT_F32 ? 3ll * c.E : c.E) || !fits(c.R > c.V ? c.R : c.V, c.E, 1 << 16)) {
        set_error("%s: rows=%d width=%d vocabulary=%d too large", what, c.R, c.E, c.V);
        return ICAP_ERR_LIMIT;
    }
    return ICAP_OK;
}

}  // namespace lce

static long long plan_bytes(int dtype, const lce::Call& c, bool any) {
    if (c.R <= 0 || c.E <= 0 || c.V <= 0) return 0;
    if (dtype == DT_F32) return lce::Plan<float>(c, nullptr, any).bytes;
    return lce::Plan<_Float16>(c, nullptr, any).bytes;
}

long long linear_ce_ws_bytes(int dtype, int R, int E, int V, int backward) {
    return plan_bytes(dtype, lce::Call{nullptr, nullptr, nullptr, E, E, nullptr, R, E, V, 0, backward ? 7 : 0}, true);
}

long long linear_ce_ws_bytes_for(int dtype, const void* h, long long ld_h, const void* w, long long ld_w, int R, int E, int V, int need) {
    return plan_bytes(dtype, lce::Call{h, w, nullptr, ld_h, ld_w, nullptr, R, E, V, 0, need & 7}, false);
}

long long linear_ce_out_floats(int dtype, int R, int V) { return R <= 0 || V <= 0 ? 0 : lce::out_floats(dtype, R, V); }

int linear_ce_fwd(int dtype, const void* h, long long ld_h, const void* w, long long ld_w, const void* bias, const long long* targets, int R, int E,
                  int V, long long ignore, int mean_over_valid, float* row_loss, float* row_lse, float* loss, float* out, void* ws, long long ws_bytes,
                  hipStream_t st) {
    const lce::Call c{h, w, bias, ld_h, ld_w, targets, R, E, V, ignore};
    if (int rc = lce::check(dtype, c, "linear_ce_fwd")) return rc;
    if (!row_loss || !row_lse || !out || !aligned16(out) || !ws || !aligned16(ws) || ws_bytes < plan_bytes(dtype, c, false)) {
        set_error("linear_ce_fwd: null result, results or a workspace that are unaligned, or a workspace that is null or too small");
        return ICAP_ERR_ARG;
    }
    if (dtype == DT_F32) return lce::fwd<float>(c, mean_over_valid, row_loss, row_lse, loss, out, (char*)ws, st);
    if (dtype == DT_BF16) return lce::fwd<__bf16>(c, mean_over_valid, row_loss, row_lse, loss, out, (char*)ws, st);
    return lce::fwd<_Float16>(c, mean_over_valid, row_loss, row_lse, loss, out, (char*)ws, st);
}

int linear_ce_bwd(int dtype, const void* h, long long ld_h, const void* w, long long ld_w, const void* bias, const long long* targets, int R, int E,
                  int V, long long ignore, const float* row_lse, const float* meta, const float* grad_out, void* dh, void* dw, void* db, void* ws,
                  long long ws_bytes, hipStream_t st) {
    const lce::Call c{h, w, bias, ld_h, ld_w, targets, R, E, V, ignore, (dh ? lce::NEED_DH : 0) | (dw ? lce::NEED_DW : 0) | (db ? lce::NEED_DB : 0)};
    if (int rc = lce::check(dtype, c, "linear_ce_bwd")) return rc;
    if (c.need == 0) return ICAP_OK;
    if (!row_lse || !meta || !aligned16(meta) || !grad_out || !ws || !aligned16(ws) || ws_bytes < plan_bytes(dtype, c, false)) {
        set_error("linear_ce_bwd: null tensor, or a workspace that is null, unaligned or too small");
        return ICAP_ERR_ARG;
    }
    if (dh && !aligned16(dh)) { set_error("linear_ce_bwd: dhidden must be 16-byte aligned"); return ICAP_ERR_ALIGN; }
    if (dw && !aligned16(dw)) { set_error("linear_ce_bwd: dweight must be 16-byte aligned"); return ICAP_ERR_ALIGN; }
    if (dtype == DT_F32) return lce::bwd<float>(c, row_lse, meta, grad_out, dh, dw, db, (char*)ws, st);
    if (dtype == DT_BF16) return lce::bwd<__bf16>(c, row_lse, meta, grad_out, dh, dw, db, (char*)ws, st);
    return lce::bwd<_Float16>(c, row_lse, meta, grad_out, dh, dw, db, (char*)ws, st);
}

}  // namespace icap
