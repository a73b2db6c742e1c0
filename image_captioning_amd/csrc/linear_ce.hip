// Softmax cross entropy of a Linear layer over a large vocabulary without its [rows, V] logits in memory:
//   x = h W^T + b,  lse_r = log sum_v exp x_rv,  loss_r = lse_r - x_r,target,  loss = scale sum_r loss_r
//   D = softmax(x) - onehot(target) (zero rows where ignored),  dh = g D W,  dW = g D^T h,  db = g sum_r D,  g = grad_out scale
// Forward: one GEMM whose epilogue keeps, of every 64-column strip of a row, only its maximum and its sum of exponentials
// (8 bytes for 64 logits) and the target's logit; a second launch joins the strips.
// Backward: the vocabulary in pieces.  The logits of a piece are formed again, turned into D in the epilogue (16 bits, row-major
// and transposed), and multiplied while the cache still holds them; dh collects the pieces in fp32.  The bias gradient is summed
// from the unrounded D.  Every sum has a fixed order.
// All products are one GEMM kernel: C[m][n] = sum_k A[m][k] B[n][k] on the 16-bit matrix cores, fp32 accumulation, operands with
// contiguous k (dh and dW take W, h and D transposed: W and h are turned once a call, D is written both ways).
//   bf16: D is rounded to bf16 (2^-9 of each value, as much as the result's own rounding).
//   fp16: D 2^14 is rounded to fp16, so that a probability of 1e-8 still has full precision; the factor leaves again exactly.
//   fp32: every operand is the sum of two fp16 values (22 bits), scaled by a power of two so that its largest magnitude is near
//   2^14; the products hi hi + hi lo + lo hi drop 2^-22 of each term: as exact as an fp32 dot product, at three fp16
//   products for one (the fp32 matrix instruction takes sixteen times a 16-bit product).
// Bound: the matrix cores (2 R E V flops a product; one forward, three backward of which the logits are repeated).
#include "packed.hpp"

namespace icap {
namespace lce {

constexpr int BK = 64, ROWB = BK * 2;               // K tile; bytes of an LDS row
constexpr int STRIP = 64;                           // columns that share one (maximum, sum) pair
constexpr float D_SCALE = 16384.0f;                 // fp16 D
constexpr float LOG2E = 1.4426950408889634f;

enum Epilogue { EP_LSE, EP_GRAD, EP_OUT };

struct Gemm {
    const unsigned short *a0, *a1, *b0, *b1;        // planes: high and (fp32 tensors) low parts
    long long lda, ldb;
    int M, N, K, pairs, ksplit, tiles_m, tiles_n;   // K % 64 == 0; pairs 1 or 3
    const float* unscale;                           // one factor on the accumulators in device memory, or null
    // EP_LSE and EP_GRAD
    const void* bias;                               // type of the tensors
    const long long* targets;
    long long ignore;
    int V, v0;                                      // column 0 of this product is word v0; words end at V
    float2* part; int strips; float* target_logit;  // EP_LSE
    const float* lse;                               // EP_GRAD
    unsigned short *d0, *d1, *t0, *t1;              // D [M][ldd] and D^T [N][ldt], planes
    long long ldd, ldt;
    int rows_pad, cols_pad;                         // D is written (zeros) up to these multiples of 64
    float* colpart; long long ldc;                  // [row blocks][ldc]
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

__device__ __forceinline__ float final_factor(const Gemm& p) {
    float f = p.f;
    if (p.f0) f *= *p.f0;
    if (p.f1) f *= *p.f1;
    if (p.f2) f *= *p.f2;
    return f;
}

// high and low 16-bit parts of a value
template <typename E>
__device__ __forceinline__ void split(float x, E& hi, E& lo) {
    hi = (E)x;
    lo = (E)(x - (float)hi);
}

template <int BM, int BN> constexpr int smem_bytes() { return 2 * (BM + BN) * ROWB; }

// WM x WN waves, each (BM / WM) x 64 of the tile.  Operands go global -> LDS without passing a register (16 bytes a lane, one wave
// 1 KB); the next K tile is in flight while the current one multiplies; one wait and one barrier a K tile.  The 16-byte slot a lane
// fetches is permuted by its row, and the fragment reads apply the same permutation, so that 16 rows meet 16 different slots.
template <typename E, typename T, int BM, int BN, int WM, int WN, int EP>
__global__ __launch_bounds__(WM * WN * 64) void gemm_kernel(const Gemm p) {
    constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, RM = TM / 32, RN = TN / 32, RPP = NW * 8;
    static_assert(TN == STRIP && TM % 32 == 0 && BM % RPP == 0 && BN % RPP == 0, "wave tiles");
    constexpr int APT = BM / RPP, BPT = BN / RPP, A_BYTES = BM * ROWB, STAGE = (BM + BN) * ROWB, EP_LD = TN + 4;
    static_assert(NW * 32 * EP_LD * 4 <= 2 * STAGE, "the waves' result images fit the staging buffers");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave - wm * WN, lr = lane & 31, lh = lane >> 5;

    // each XCD (workgroups go round them) walks a contiguous range of tiles, in which neighbours share their B panel
    const int nwg = gridDim.x, xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, tq = nwg >> 3, tr = nwg & 7;
    const int tlin = xcd * tq + (xcd < tr ? xcd : tr) + slot;
    const int tile_n = tlin / p.tiles_m, tile_m = tlin - tile_n * p.tiles_m;
    const int m0 = tile_m * BM, n0 = tile_n * BN;

    const int srow = wave * 8 + (lane >> 3), lslot = (lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7);
    long long a_off[APT], b_off[BPT];
#pragma unroll
    for (int i = 0; i < APT; ++i) a_off[i] = (long long)min(m0 + i * RPP + srow, p.M - 1) * p.lda + 8 * lslot;
#pragma unroll
    for (int i = 0; i < BPT; ++i) b_off[i] = (long long)min(n0 + i * RPP + srow, p.N - 1) * p.ldb + 8 * lslot;
    const int nk = p.K / BK, total = nk * p.pairs;
    const int per = (total + p.ksplit - 1) / p.ksplit, t_lo = min((int)blockIdx.y * per, total), t_hi = min(t_lo + per, total);
    int pair = t_lo / nk, kt = t_lo - pair * nk;
    auto issue = [&](int buf) __attribute__((always_inline)) {
        unsigned char* base = smem + buf * STAGE + wave * 1024;
        const unsigned short* a = (pair == 2 ? p.a1 : p.a0) + (long long)kt * BK;
        const unsigned short* b = (pair == 1 ? p.b1 : p.b0) + (long long)kt * BK;
#pragma unroll
        for (int i = 0; i < APT; ++i) load16(a + a_off[i], base + i * (NW * 1024));
#pragma unroll
        for (int i = 0; i < BPT; ++i) load16(b + b_off[i], base + A_BYTES + i * (NW * 1024));
        if (++kt == nk) { kt = 0; ++pair; }
    };
    f32x16 acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int sw = (lr >> 1) & 7;
    auto compute = [&](int buf) __attribute__((always_inline)) {
        const unsigned char* sa = smem + buf * STAGE + (wm * TM + lr) * ROWB;
        const unsigned char* sb = smem + buf * STAGE + A_BYTES + (wn * TN + lr) * ROWB;
#pragma unroll
        for (int s = 0; s < BK / 16; ++s) {
            const int off = ((2 * s + lh) ^ sw) * 16;
            typename Vec<E>::x8 af[RM], bf[RN];
#pragma unroll
            for (int i = 0; i < RM; ++i) af[i] = *reinterpret_cast<const typename Vec<E>::x8*>(sa + i * 32 * ROWB + off);
#pragma unroll
            for (int j = 0; j < RN; ++j) bf[j] = *reinterpret_cast<const typename Vec<E>::x8*>(sb + j * 32 * ROWB + off);
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < RN; ++j) acc[i][j] = Mma<E>::go(af[i], bf[j], acc[i][j]);
        }
    };
    if (t_lo < t_hi) issue(0);
    for (int t = t_lo; t < t_hi; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();           // K tile t is there for every wave, and everybody has left the buffer filled next
        asm volatile("" ::: "memory");
        if (t + 1 < t_hi) issue((t + 1 - t_lo) & 1);
        compute((t - t_lo) & 1);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // epilogue, every wave on its own, 32 rows at a time: accumulators -> the wave's image in LDS -> eight columns a lane, eight lanes a row
    float* ew = reinterpret_cast<float*>(smem) + wave * 32 * EP_LD;
    const float un = p.unscale ? *p.unscale : 1.0f;
    const float ff = EP == EP_OUT ? (p.acc ? 1.0f : final_factor(p)) : 1.0f;
    const int c8 = lane & 7, n = n0 + wn * TN + 8 * c8;         // this lane's first column
    float bias[8], colsum[8];
    if constexpr (EP != EP_OUT) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            colsum[e] = 0.f;
            bias[e] = (p.bias && n + e < p.N) ? (float)((const T*)p.bias)[p.v0 + n + e] : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) ew[((e & 3) + 8 * (e >> 2) + 4 * lh) * EP_LD + j * 32 + lr] = acc[i][j][e];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = q * 8 + (lane >> 3), m = m0 + wm * TM + i * 32 + row;
            float* im = ew + row * EP_LD + 8 * c8;
            const f32x4 x0 = *reinterpret_cast<const f32x4*>(im), x1 = *reinterpret_cast<const f32x4*>(im + 4);
            float v[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
            if constexpr (EP == EP_LSE) {
                const long long t = m < p.M ? p.targets[m] - p.v0 : -1;
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = n + e < p.N ? fmaf(v[e], un, bias[e]) : -INFINITY;
                    mx = fmaxf(mx, v[e]);
                    if (t == n + e && n + e < p.N) p.target_logit[m] = v[e];
                }
                mx = fmaxf(mx, dpp_f<DPP_QUAD_SWAP1>(mx));
                mx = fmaxf(mx, dpp_f<DPP_QUAD_SWAP2>(mx));
                mx = fmaxf(mx, dpp_f<DPP_HALF_MIRROR>(mx));
                const float base = mx == -INFINITY ? 0.f : mx;
                float s = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) s += __builtin_amdgcn_exp2f((v[e] - base) * LOG2E);
                s += dpp_f<DPP_QUAD_SWAP1>(s);
                s += dpp_f<DPP_QUAD_SWAP2>(s);
                s += dpp_f<DPP_HALF_MIRROR>(s);
                const int strip = tile_n * WN + wn;
                if (c8 == 0 && m < p.M && strip < p.strips) p.part[(long long)m * p.strips + strip] = make_float2(mx, s);
            } else if constexpr (EP == EP_GRAD) {
                const int mm = min(m, p.M - 1);
                const long long tg = p.targets[mm];
                const bool on = m < p.M && tg >= 0 && tg < p.V && tg != p.ignore;
                const float lse = p.lse[mm];
                const long long t = tg - p.v0;
                typename Vec<E>::x8 hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float d = __builtin_amdgcn_exp2f((fmaf(v[e], un, bias[e]) - lse) * LOG2E);
                    if (t == n + e) d -= 1.0f;
                    d = (on && n + e < p.N) ? d : 0.f;
                    colsum[e] += d;
                    if constexpr (sizeof(E) == 2 && !__is_same(E, __bf16)) d *= D_SCALE;
                    v[e] = d;
                    E h, l;
                    split<E>(d, h, l);
                    hi[e] = h;
                    lo[e] = l;
                }
                if (m < p.M && n < p.cols_pad) {
                    *reinterpret_cast<typename Vec<E>::x8*>(p.d0 + (long long)m * p.ldd + n) = hi;
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<typename Vec<E>::x8*>(p.d1 + (long long)m * p.ldd + n) = lo;
                }
                *reinterpret_cast<f32x4*>(im) = f32x4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<f32x4*>(im + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                if (m < p.M && n < p.N) {
                    if (p.acc) {
                        float* o = p.acc + ((long long)blockIdx.y * p.M + m) * p.N + n;
                        if (p.N % 4 == 0 && n + 8 <= p.N) {
                            f32x4 y0 = x0, y1 = x1;
                            if (p.accumulate) { y0 += *reinterpret_cast<const f32x4*>(o); y1 += *reinterpret_cast<const f32x4*>(o + 4); }
                            *reinterpret_cast<f32x4*>(o) = y0;
                            *reinterpret_cast<f32x4*>(o + 4) = y1;
                        } else {
                            for (int e = 0; e < 8 && n + e < p.N; ++e) o[e] = p.accumulate ? o[e] + v[e] : v[e];
                        }
                    } else {
                        T* o = (T*)p.out + (long long)m * p.ldo + n;
                        if (p.ldo % 8 == 0 && n + 8 <= p.N) {
                            typename Vec<T>::x8 y;
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[e] = (T)(v[e] * ff);
                            *reinterpret_cast<typename Vec<T>::x8*>(o) = y;
                        } else {
                            for (int e = 0; e < 8 && n + e < p.N; ++e) o[e] = (T)(v[e] * ff);
                        }
                    }
                }
            }
        }
        if constexpr (EP == EP_GRAD) {
            // the same 32 rows transposed: a lane takes a column
            const int nn = n0 + wn * TN + lane, mb = m0 + wm * TM + i * 32;
            if (nn < p.N && mb < p.rows_pad) {
#pragma unroll
                for (int r8 = 0; r8 < 4; ++r8) {
                    typename Vec<E>::x8 hi, lo;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        E h, l;
                        split<E>(ew[(r8 * 8 + e) * EP_LD + lane], h, l);
                        hi[e] = h;
                        lo[e] = l;
                    }
                    *reinterpret_cast<typename Vec<E>::x8*>(p.t0 + (long long)nn * p.ldt + mb + r8 * 8) = hi;
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<typename Vec<E>::x8*>(p.t1 + (long long)nn * p.ldt + mb + r8 * 8) = lo;
                }
            }
        }
    }
    if constexpr (EP == EP_GRAD) {
        if (p.colpart) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                colsum[e] += __shfl_xor(colsum[e], 8);
                colsum[e] += __shfl_xor(colsum[e], 16);
                colsum[e] += __shfl_xor(colsum[e], 32);
                if (lane < 8 && n + e < p.N) p.colpart[(long long)(tile_m * WM + wm) * p.ldc + p.v0 + n + e] = colsum[e];
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

// loss (its sum in 64 bits) and the scale of every row
__global__ __launch_bounds__(1024) void loss_kernel(const float* row_loss, const long long* targets, int R, int V, long long ignore, int mean_over_valid,
                                                    float* out) {
    __shared__ double ss[16];
    __shared__ int sc[16];
    double s = 0.0;
    int c = 0;
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
        out[1] = over > 0 ? 1.0f / (float)over : 0.f;
    }
}

// ------------------------------------------------------------------------------------------------ operands
// largest magnitude of a matrix: one value a workgroup
__global__ __launch_bounds__(256) void amax_kernel(const float* x, long long ld, int R, int C, float* part) {
    float m = 0.f;
    for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < R; r += gridDim.x * 4)
        for (int c = threadIdx.x & 63; c < C; c += 64) m = fmaxf(m, fabsf(x[r * ld + c]));
    __shared__ float red[4];
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
constexpr int AMAX_WGS = 256;

// scales[0..3] = 2^s_h, 2^-s_h, 2^s_w, 2^-s_w, scales[4] = 2^-(s_h + s_w): powers of two that bring the largest magnitude to [2^13, 2^14]
__global__ __launch_bounds__(256) void scales_kernel(const float* part_h, const float* part_w, float* scales) {
    __shared__ float red[2][4];
    const int wave = threadIdx.x >> 6;
    const float h = wave_max(part_h[threadIdx.x]), w = wave_max(part_w[threadIdx.x]);
    if ((threadIdx.x & 63) == 0) { red[0][wave] = h; red[1][wave] = w; }
    __syncthreads();
    if (threadIdx.x < 2) {
        const float m = fmaxf(fmaxf(red[threadIdx.x][0], red[threadIdx.x][1]), fmaxf(red[threadIdx.x][2], red[threadIdx.x][3]));
        int e = 0;
        if (m > 0.f && m < INFINITY) e = 14 - min(max(ilogbf(m) + 1, -46), 74);     // 2^+-60: both factors and their product stay fp32 values
        scales[2 * threadIdx.x] = ldexpf(1.0f, e);
        scales[2 * threadIdx.x + 1] = ldexpf(1.0f, -e);
    }
    __syncthreads();
    if (threadIdx.x == 0) scales[4] = scales[1] * scales[3];
}

// src [R][C] (rows ld apart) -> 16-bit planes of it: rows [R][Cp] and / or transposed [C][Rp], zeros up to Cp and Rp (multiples of 64)
template <typename T, typename E>
__global__ __launch_bounds__(256) void planes_kernel(const T* src, long long ld, int R, int C, int Rp, int Cp, const float* scale, E* r0, E* r1,
                                                     E* c0, E* c1) {
    __shared__ E hi[64][66];
    __shared__ E lo[64][66];
    const int cx = blockIdx.x * 64, ry = blockIdx.y * 64, tid = threadIdx.x;
    const float f = scale ? *scale : 1.0f;
    for (int i = tid; i < 64 * 64; i += 256) {
        const int r = i >> 6, c = i & 63;
        float x = 0.f;
        if (ry + r < R && cx + c < C) x = (float)src[(long long)(ry + r) * ld + cx + c] * f;
        E h, l;
        split<E>(x, h, l);
        hi[r][c] = h;
        if constexpr (sizeof(T) == 4) lo[r][c] = l;
        if (r0 && ry + r < R) {
            r0[(long long)(ry + r) * Cp + cx + c] = h;
            if constexpr (sizeof(T) == 4) r1[(long long)(ry + r) * Cp + cx + c] = l;
        }
    }
    if (!c0) return;
    __syncthreads();
    for (int i = tid; i < 64 * 64; i += 256) {
        const int c = i >> 6, r = i & 63;
        if (cx + c < C) {
            c0[(long long)(cx + c) * Rp + ry + r] = hi[r][c];
            if constexpr (sizeof(T) == 4) c1[(long long)(cx + c) * Rp + ry + r] = lo[r][c];
        }
    }
}

// out[i] = factor * sum over splits of acc[split][i], in order
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float* acc, int splits, long long n, T* out, const Gemm p) {
    const float f = final_factor(p);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = acc[i];
        for (int z = 1; z < splits; ++z) s += acc[z * n + i];
        out[i] = (T)(s * f);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void bias_kernel(const float* colpart, int blocks, int V, T* out, const float* f0, const float* f1) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= V) return;
    float s = 0.f;
    for (int b = 0; b < blocks; ++b) s += colpart[(long long)b * V + v];
    out[v] = (T)(s * (*f0 * *f1));
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

// a tile of 256 x 256 when there are enough of them for the 256 CUs, of 128 x 128 (two workgroups a CU) otherwise
struct Shape { bool big; int tiles_m, tiles_n; };
inline Shape shape_of(int M, int N) {
    const long long big = up(M, 256) / 256 * (up(N, 256) / 256);
    const bool b = big >= 192;
    const int t = b ? 256 : 128;
    return {b, (int)(up(M, t) / t), (int)(up(N, t) / t)};
}
inline Shape resized(const Shape& s, int M, int N) { const int t = s.big ? 256 : 128; return {s.big, (int)(up(M, t) / t), (int)(up(N, t) / t)}; }
// few tiles: the contraction in pieces of at least four K tiles, up to two workgroups a CU
inline int splits_of(const Shape& s, long long ktiles) {
    const long long tiles = (long long)s.tiles_m * s.tiles_n, want = s.big ? 256 : 512;
    long long k = (want + tiles / 2) / tiles;
    if (k > ktiles / 4) k = ktiles / 4;
    return (int)(k < 1 ? 1 : (k > 32 ? 32 : k));
}

template <typename E, typename T, int BM, int BN, int WM, int WN, int EP>
int go(const Gemm& p, hipStream_t st) {
    static const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_kernel<E, T, BM, BN, WM, WN, EP>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<BM, BN>());
    if (rc != hipSuccess) { set_error("linear_ce: cannot raise the dynamic LDS limit: %s", hipGetErrorString(rc)); return ICAP_ERR_HIP_BASE + (int)rc; }
    hipLaunchKernelGGL((gemm_kernel<E, T, BM, BN, WM, WN, EP>), dim3((unsigned)(p.tiles_m * p.tiles_n), p.ksplit), dim3(WM * WN * 64),
                       (smem_bytes<BM, BN>()), st, p);
    return launch_status("linear_ce");
}

template <typename E, typename T, int EP>
int gemm(Gemm& p, const Shape& s, hipStream_t st) {
    p.tiles_m = s.tiles_m;
    p.tiles_n = s.tiles_n;
    return s.big ? go<E, T, 256, 256, 2, 4, EP>(p, st) : go<E, T, 128, 128, 2, 2, EP>(p, st);
}

struct Call {
    const void *h, *w, *bias;
    long long ld_h, ld_w;
    const long long* targets;
    int R, E, V;
    long long ignore;
};

// bytes of D and D^T that a piece of the vocabulary may take: what the last-level cache holds beside its operands
constexpr long long PIECE_BYTES = 256ll << 20;

template <typename T> struct Of { typedef T E; static constexpr int planes = 1; };
template <> struct Of<float> { typedef _Float16 E; static constexpr int planes = 2; };

// whether a matrix can be read by the GEMM as it is: 16 bits, rows of whole 64-value K tiles, 16-byte pieces
template <typename T>
bool direct(const void* x, long long ld, int C) { return sizeof(T) == 2 && C % 64 == 0 && ld % 8 == 0 && aligned16(x); }

template <typename T>
struct Operand {
    typename Of<T>::E *row0 = nullptr, *row1 = nullptr, *col0 = nullptr, *col1 = nullptr;
    long long ld = 0, ldc = 0;
};

// room for the planes of a matrix (want_rows: as the GEMM's A or B in the logits; want_cols: transposed)
template <typename T>
Operand<T> room(Space& ws, const void* x, long long ld, int R, int C, bool want_cols, bool is_direct) {
    typedef typename Of<T>::E E;
    Operand<T> o;
    o.ld = up(C, 64);
    o.ldc = up(R, 64);
    if (is_direct) { o.row0 = (E*)const_cast<void*>(x); o.ld = ld; }
    else {
        o.row0 = ws.take<E>(R * o.ld);
        if (Of<T>::planes == 2) o.row1 = ws.take<E>(R * o.ld);
    }
    if (want_cols) {
        o.col0 = ws.take<E>(C * o.ldc);
        if (Of<T>::planes == 2) o.col1 = ws.take<E>(C * o.ldc);
    }
    return o;
}

template <typename T>
void fill(const Operand<T>& o, const void* x, long long ld, int R, int C, bool is_direct, const float* scale, hipStream_t st) {
    typedef typename Of<T>::E E;
    if (is_direct && !o.col0) return;
    hipLaunchKernelGGL((planes_kernel<T, E>), dim3((unsigned)(up(C, 64) / 64), (unsigned)(up(R, 64) / 64)), dim3(256), 0, st, (const T*)x, ld, R, C,
                       (int)up(R, 64), (int)up(C, 64), scale, is_direct ? (E*)nullptr : o.row0, o.row1, o.col0, o.col1);
}

template <typename T>
struct Plan {
    bool dh_direct, dw_direct;
    Operand<T> h, w;
    float *scales, *amax;
    // forward
    float2* part; float* target_logit; int strips;
    // backward
    int piece; long long ldd, ldt;
    typename Of<T>::E *d0, *d1, *t0, *t1;
    float *colpart, *acc_h, *acc_w;
    Shape s_logit, s_h, s_w; int k_h, k_w;
    long long bytes;

    Plan(const Call& c, bool backward, char* base) {
        typedef typename Of<T>::E E;
        Space ws{base};
        dh_direct = direct<T>(c.h, c.ld_h, c.E);
        dw_direct = direct<T>(c.w, c.ld_w, c.E);
        if (!base) dh_direct = dw_direct = false;           // the size is asked for without pointers: the larger of the two
        h = room<T>(ws, c.h, c.ld_h, c.R, c.E, backward, dh_direct);
        w = room<T>(ws, c.w, c.ld_w, c.V, c.E, backward, dw_direct);
        scales = ws.take<float>(8);
        amax = ws.take<float>(2 * AMAX_WGS);
        if (!backward) {
            strips = (int)(up(c.V, STRIP) / STRIP);
            part = ws.take<float2>((long long)c.R * strips);
            target_logit = ws.take<float>(c.R);
        } else {
            const long long rp = up(c.R, 64);
            long long v = PIECE_BYTES / (2 * rp * 2 * Of<T>::planes) / 256 * 256;
            if (v < 256) v = 256;
            if (v >= c.V) v = c.V;
            else v = up((c.V + (c.V + v - 1) / v - 1) / ((c.V + v - 1) / v), 256);      // pieces of about the same size
            piece = (int)v;
            ldd = up(piece, 64);
            ldt = rp;
            d0 = ws.take<E>(c.R * ldd);
            t0 = ws.take<E>(piece * ldt);
            d1 = t1 = nullptr;
            if (Of<T>::planes == 2) { d1 = ws.take<E>(c.R * ldd); t1 = ws.take<E>(piece * ldt); }
            const int pairs = Of<T>::planes == 2 ? 3 : 1;
            s_logit = shape_of(c.R, piece);
            s_h = shape_of(c.R, c.E);
            s_w = shape_of(piece, c.E);
            k_h = splits_of(s_h, ldd / 64 * pairs);
            k_w = splits_of(s_w, ldt / 64 * pairs);
            colpart = ws.take<float>((long long)s_logit.tiles_m * 2 * c.V);
            acc_h = ws.take<float>((k_h > 1 || piece < c.V) ? (long long)k_h * c.R * c.E : 0);
            acc_w = ws.take<float>(k_w > 1 ? (long long)k_w * piece * c.E : 0);
        }
        bytes = ws.at;
    }
};

template <typename T>
void operands(const Call& c, Plan<T>& p, hipStream_t st) {
    const float *sh = nullptr, *sw = nullptr;
    if constexpr (sizeof(T) == 4) {
        hipLaunchKernelGGL(amax_kernel, dim3(AMAX_WGS), dim3(256), 0, st, (const float*)c.h, c.ld_h, c.R, c.E, p.amax);
        hipLaunchKernelGGL(amax_kernel, dim3(AMAX_WGS), dim3(256), 0, st, (const float*)c.w, c.ld_w, c.V, c.E, p.amax + AMAX_WGS);
        hipLaunchKernelGGL(scales_kernel, dim3(1), dim3(256), 0, st, p.amax, p.amax + AMAX_WGS, p.scales);
        sh = p.scales;
        sw = p.scales + 2;
    }
    fill<T>(p.h, c.h, c.ld_h, c.R, c.E, p.dh_direct, sh, st);
    fill<T>(p.w, c.w, c.ld_w, c.V, c.E, p.dw_direct, sw, st);
}

template <typename T>
Gemm logits(const Call& c, const Plan<T>& p, int v0, int vn) {
    Gemm g{};
    g.a0 = (const unsigned short*)p.h.row0;
    g.a1 = (const unsigned short*)p.h.row1;
    g.b0 = (const unsigned short*)p.w.row0 + v0 * p.w.ld;
    g.b1 = p.w.row1 ? (const unsigned short*)p.w.row1 + v0 * p.w.ld : nullptr;
    g.lda = p.h.ld;
    g.ldb = p.w.ld;
    g.M = c.R; g.N = vn; g.K = (int)up(c.E, 64);
    g.pairs = Of<T>::planes == 2 ? 3 : 1;
    g.ksplit = 1;
    g.unscale = sizeof(T) == 4 ? p.scales + 4 : nullptr;
    g.bias = c.bias; g.targets = c.targets; g.ignore = c.ignore; g.V = c.V; g.v0 = v0;
    return g;
}

template <typename T>
int fwd(const Call& c, int mean_over_valid, float* row_loss, float* row_lse, float* out, char* ws, hipStream_t st) {
    typedef typename Of<T>::E E;
    Plan<T> p(c, false, ws);
    operands<T>(c, p, st);
    Gemm g = logits<T>(c, p, 0, c.V);
    g.part = p.part; g.strips = p.strips; g.target_logit = p.target_logit;
    if (int rc = gemm<E, T, EP_LSE>(g, shape_of(c.R, c.V), st)) return rc;
    hipLaunchKernelGGL(lse_kernel, dim3((c.R + 3) / 4), dim3(256), 0, st, p.part, p.strips, p.target_logit, c.targets, c.R, c.V, c.ignore, row_loss, row_lse);
    hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, row_loss, c.targets, c.R, c.V, c.ignore, mean_over_valid, out);
    return launch_status("linear_ce_fwd");
}

template <typename T>
int bwd(const Call& c, const float* row_lse, const float* meta, const float* grad_out, void* dh, void* dw, void* db, char* ws, hipStream_t st) {
    typedef typename Of<T>::E E;
    Plan<T> p(c, true, ws);
    operands<T>(c, p, st);
    const float back = __is_same(E, _Float16) ? 1.0f / D_SCALE : 1.0f;
    for (int v0 = 0; v0 < c.V; v0 += p.piece) {
        const int vn = c.V - v0 < p.piece ? c.V - v0 : p.piece;
        Gemm g = logits<T>(c, p, v0, vn);
        g.lse = row_lse;
        g.d0 = (unsigned short*)p.d0; g.d1 = (unsigned short*)p.d1; g.t0 = (unsigned short*)p.t0; g.t1 = (unsigned short*)p.t1;
        g.ldd = p.ldd; g.ldt = p.ldt;
        g.rows_pad = (int)up(c.R, 64); g.cols_pad = (int)up(vn, 64);
        g.colpart = db ? p.colpart : nullptr; g.ldc = c.V;
        if (int rc = gemm<E, T, EP_GRAD>(g, resized(p.s_logit, c.R, vn), st)) return rc;
        if (dh) {
            Gemm q{};
            q.a0 = (const unsigned short*)p.d0; q.a1 = (const unsigned short*)p.d1;
            q.b0 = (const unsigned short*)p.w.col0 + v0; q.b1 = p.w.col1 ? (const unsigned short*)p.w.col1 + v0 : nullptr;
            q.lda = p.ldd; q.ldb = p.w.ldc;
            q.M = c.R; q.N = c.E; q.K = (int)up(vn, 64);
            q.pairs = g.pairs;
            q.ksplit = p.k_h;
            q.f0 = grad_out; q.f1 = meta + 1; q.f2 = sizeof(T) == 4 ? p.scales + 3 : nullptr; q.f = back;
            const bool whole = p.k_h == 1 && p.piece >= c.V;
            if (whole) { q.out = dh; q.ldo = c.E; }
            else { q.acc = p.acc_h; q.accumulate = v0 > 0; }
            if (int rc = gemm<E, T, EP_OUT>(q, p.s_h, st)) return rc;
            if (!whole && v0 + vn == c.V) {
                const long long n = (long long)c.R * c.E;
                hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(up(n, 1024) / 1024 > 4096 ? 4096 : up(n, 1024) / 1024)), dim3(256), 0, st, p.acc_h, p.k_h, n,
                                   (T*)dh, q);
            }
        }
        if (dw) {
            Gemm q{};
            q.a0 = (const unsigned short*)p.t0; q.a1 = (const unsigned short*)p.t1;
            q.b0 = (const unsigned short*)p.h.col0; q.b1 = (const unsigned short*)p.h.col1;
            q.lda = p.ldt; q.ldb = p.h.ldc;
            q.M = vn; q.N = c.E; q.K = (int)up(c.R, 64);
            q.pairs = g.pairs;
            q.ksplit = p.k_w;
            q.f0 = grad_out; q.f1 = meta + 1; q.f2 = sizeof(T) == 4 ? p.scales + 1 : nullptr; q.f = back;
            T* dst = (T*)dw + (long long)v0 * c.E;
            if (p.k_w == 1) { q.out = dst; q.ldo = c.E; }
            else q.acc = p.acc_w;
            if (int rc = gemm<E, T, EP_OUT>(q, resized(p.s_w, vn, c.E), st)) return rc;
            if (p.k_w > 1) {
                const long long n = (long long)vn * c.E;
                hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(up(n, 1024) / 1024 > 4096 ? 4096 : up(n, 1024) / 1024)), dim3(256), 0, st, p.acc_w, p.k_w, n, dst, q);
            }
        }
    }
    if (db)
        hipLaunchKernelGGL((bias_kernel<T>), dim3((c.V + 255) / 256), dim3(256), 0, st, p.colpart, p.s_logit.tiles_m * 2, c.V, (T*)db, grad_out, meta + 1);
    return launch_status("linear_ce_bwd");
}

static int check(int dtype, const Call& c, const char* what) {
    if (dtype < 0 || dtype > 2) { set_error("%s: unknown type %d", what, dtype); return ICAP_ERR_ARG; }
    if (!c.h || !c.w || !c.targets || c.R <= 0 || c.E <= 0 || c.V <= 0 || c.ld_h < c.E || c.ld_w < c.E) {
        set_error("%s: null tensor, empty size or overlapping rows", what);
        return ICAP_ERR_ARG;
    }
    // blocks of 64 rows are a grid's second index, tiles are counted in 32 bits
    if (c.R > 65535 * 64 || c.E > (1 << 20) || c.V > 65535 * 64 || up(c.R, 128) / 128 * (up(c.V, 128) / 128) > 0x7fffffffLL) {
        set_error("%s: rows=%d width=%d vocabulary=%d too large", what, c.R, c.E, c.V);
        return ICAP_ERR_LIMIT;
    }
    return ICAP_OK;
}

}  // namespace lce

long long linear_ce_ws_bytes(int dtype, int R, int E, int V, int backward) {
    lce::Call c{nullptr, nullptr, nullptr, E, E, nullptr, R, E, V, 0};
    if (R <= 0 || E <= 0 || V <= 0) return 0;
    if (dtype == DT_F32) return lce::Plan<float>(c, backward, nullptr).bytes;
    return lce::Plan<_Float16>(c, backward, nullptr).bytes;
}

int linear_ce_fwd(int dtype, const void* h, long long ld_h, const void* w, long long ld_w, const void* bias, const long long* targets, int R, int E,
                  int V, long long ignore, int mean_over_valid, float* row_loss, float* row_lse, float* out, void* ws, long long ws_bytes,
                  hipStream_t st) {
    const lce::Call c{h, w, bias, ld_h, ld_w, targets, R, E, V, ignore};
    if (int rc = lce::check(dtype, c, "linear_ce_fwd")) return rc;
    if (!row_loss || !row_lse || !out || !ws || !aligned16(ws) || ws_bytes < linear_ce_ws_bytes(dtype, R, E, V, 0)) {
        set_error("linear_ce_fwd: null result, or a workspace that is null, unaligned or too small");
        return ICAP_ERR_ARG;
    }
    if (dtype == DT_F32) return lce::fwd<float>(c, mean_over_valid, row_loss, row_lse, out, (char*)ws, st);
    if (dtype == DT_BF16) return lce::fwd<__bf16>(c, mean_over_valid, row_loss, row_lse, out, (char*)ws, st);
    return lce::fwd<_Float16>(c, mean_over_valid, row_loss, row_lse, out, (char*)ws, st);
}

int linear_ce_bwd(int dtype, const void* h, long long ld_h, const void* w, long long ld_w, const void* bias, const long long* targets, int R, int E,
                  int V, long long ignore, const float* row_lse, const float* meta, const float* grad_out, void* dh, void* dw, void* db, void* ws,
                  long long ws_bytes, hipStream_t st) {
    const lce::Call c{h, w, bias, ld_h, ld_w, targets, R, E, V, ignore};
    if (int rc = lce::check(dtype, c, "linear_ce_bwd")) return rc;
    if (!row_lse || !meta || !grad_out || !ws || !aligned16(ws) || ws_bytes < linear_ce_ws_bytes(dtype, R, E, V, 1)) {
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
