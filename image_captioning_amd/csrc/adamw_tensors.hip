// AdamW over many tensors where they lie: one launch takes up to AT_MAX of them, their pointers in the kernel's arguments (no
// table in device memory to build, copy or keep, and a captured launch holds everything it needs).  The update is the one of
// adamw_kernel (train.hip), in fp32 whatever the parameters' type, rounded once into it:
//   m += (g - m) (1 - b1);  v = v b2 + g g (1 - b2);  p = p (1 - lr wd) - (m / (sqrt(v) / sqrt(1 - b2^t) + eps)) lr / (1 - b1^t)
// States in 32 bits are fp32 tensors.  States in 8 bits are e4m3 codes with one fp32 scale for every 256 values of a tensor (scale =
// largest magnitude / 448):
//   * m is rounded to nearest: it moves by (1 - b1) (g - m), 10 % of the gradient's noise a step, which is more than a code's half
//     step often enough for the noise itself to carry it on;
//   * the second moment is held as sqrt(v), which doubles the range in which small values are told apart (2^18 : 1), and is rounded at
//     random with the right mean: v b2 differs from v by 0.1 %, far less than half a code (3 - 6 %), so to nearest it would never
//     fall again.  It is the mean of sqrt(v); that of v lies above by the rounding's variance.  A value above zero never rounds to zero,
//     since m / eps would follow: below the first code, 2^-9 of the scale, it becomes that code, and the mean is higher there.
// Sixteen random bits a value come from the counter-based generator of uniform01 (seed; step and tensor; place), so a run can be
// repeated, and nothing is kept between calls.
// Bound: HBM.  3 size(p) + 16 bytes a value with 32-bit states, 3 size(p) + 4 + 1/16 with 8-bit ones.  One wave owns 256 values at a
// time (four a lane, 16 bytes of fp32), which is one scale's block: the largest magnitude is one wave reduction, no LDS, no barrier.
// Measured: 20 fp32 tensors, 15.7 M values, fp32 states 118 us = 3.7 TB/s; 48 bf16 tensors, 176 M values, 8-bit states 444 us = 4.0 TB/s (a
// large copy: 4.7); 250 fp32 tensors of 32 to 409600 values, 12.4 M in all, 8-bit states 111 us in five launches = 1.8 TB/s: 70 % of the values lie
// in tensors that are not aligned for whole loads and take the loop over single values, as up to 1024 values at every tensor's end do.
#include "packed.hpp"
#include <math.h>

namespace icap {

constexpr int AT_MAX = 62;                  // tensors a launch: 62 x 64 bytes of kernel arguments (the limit is 4096)
constexpr int AT_BLOCK = 256;               // values that share a scale
constexpr int AT_WAVE_BLOCKS = 4;           // blocks a wave owns
constexpr int AT_CHUNK = 4 * AT_WAVE_BLOCKS * AT_BLOCK;      // values a workgroup of four waves owns
constexpr unsigned AT_VEC = 1u << 31;       // in AdamTensor::index: four values can be read at once

struct AdamTensor {
    void* p; const void* g; void* m; void* v; float* ms; float* vs;
    long long n;
    unsigned first, index;                  // first workgroup; place in the caller's list
};

struct AdamTable {
    AdamTensor t[AT_MAX];
    int count, step;                        // one step for all (or what is added to *step_dev)
    float decay, one_minus_b1, b2, one_minus_b2, eps, grad_scale, step_size, inv_bc2_sqrt;
    unsigned long long seed;
    const int* step_dev;
    double lr, beta1, beta2;
};
static_assert(sizeof(AdamTable) <= 4096, "kernel arguments");

__device__ __forceinline__ unsigned long long mix64(unsigned long long z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
    return z ^ (z >> 31);
}

template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const f32x4*>(p);
    else return __builtin_convertvector(*reinterpret_cast<const typename Vec<T>::x4*>(p), f32x4);
}
template <typename T>
__device__ __forceinline__ void put4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
    else *reinterpret_cast<typename Vec<T>::x4*>(p) = __builtin_convertvector(v, typename Vec<T>::x4);
}

__device__ __forceinline__ f32x4 codes_to_f32(unsigned c) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    return f32x4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ unsigned f32_to_codes(f32x4 y) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
}

// scale of a block and what its values are multiplied with; a block below 1e-30 is all zeros
__device__ __forceinline__ void block_scale(float most, float& scale, float& inverse) {
    const bool some = !(most < 1e-30f);
    scale = some ? most * (1.0f / 448.0f) : 0.f;
    inverse = some ? (1.0f / most) * 448.0f : 0.f;
}

// y in [0, 448] to one of its two neighbours in e4m3, the upper one with the probability of the place between them
__device__ __forceinline__ float round_at_random(float y, float u, unsigned r16) {
    const float normal = __uint_as_float((__float_as_uint(y) + (r16 << 4)) & 0xFFF00000u);
    const float below = floorf(y * 512.0f + (float)r16 * (1.0f / 65536.0f)) * (1.0f / 512.0f);     // spacing 2^-9 under 2^-6
    float z = y >= 0.015625f ? normal : below;
    z = z > 448.0f ? 448.0f : z;
    return (u > 0.f && z == 0.f) ? 0.001953125f : z;
}

// the update of a lane's four values; 8-bit states come and go as codes, with the block's scales
template <int BITS>
__device__ __forceinline__ void adamw_four(const AdamTable& a, float step_size, float inv_bc2, unsigned long long key, long long place, f32x4& p, f32x4 g,
                                           f32x4& m, f32x4& v, unsigned& mc, unsigned& vc, float& ms, float& vs) {
    if constexpr (BITS == 8) {
        m = codes_to_f32(mc) * ms;
        v = codes_to_f32(vc) * vs;
        v = v * v;
    }
    f32x4 u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float gr = g[e] * a.grad_scale;
        m[e] = m[e] + (gr - m[e]) * a.one_minus_b1;
        v[e] = v[e] * a.b2 + (gr * gr) * a.one_minus_b2;
        u[e] = sqrtf(v[e]);
        const float denom = u[e] * inv_bc2 + a.eps;
        p[e] = p[e] * a.decay - (m[e] / denom) * step_size;
    }
    if constexpr (BITS == 8) {
        float most_m = 0.f, most_u = 0.f;               // places behind the tensor's end hold zeros
#pragma unroll
        for (int e = 0; e < 4; ++e) { most_m = fmaxf(most_m, fabsf(m[e])); most_u = fmaxf(most_u, u[e]); }
        float im, iu;
        block_scale(wave_max(most_m), ms, im);
        block_scale(wave_max(most_u), vs, iu);
        const unsigned long long draw = mix64(key + 0x9E3779B97F4A7C15ULL * (unsigned long long)(place >> 2));
        f32x4 ym, yu;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y = m[e] * im;
            y = y > 448.0f ? 448.0f : y;                // comparisons, not min / max: a NaN stays one
            ym[e] = y < -448.0f ? -448.0f : y;
            float z = u[e] * iu;
            z = z > 448.0f ? 448.0f : z;
            yu[e] = round_at_random(z, iu > 0.f ? u[e] : 0.f, (unsigned)(draw >> (16 * e)) & 0xFFFFu);
        }
        mc = f32_to_codes(ym);
        vc = f32_to_codes(yu);
    }
}

template <typename P, typename G, int BITS>
__global__ __launch_bounds__(256) void adamw_tensors_kernel(const AdamTable a) {
    // the tensor this workgroup belongs to: the last one that starts at or before it
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.t[mid].first <= blockIdx.x) lo = mid; else hi = mid;
    }
    const AdamTensor& t = a.t[lo];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long n = t.n, base = (long long)(blockIdx.x - t.first) * AT_CHUNK + wave * (AT_WAVE_BLOCKS * AT_BLOCK), blk = base / AT_BLOCK;
    if (base >= n) return;
    int step = a.step;
    float step_size = a.step_size, inv_bc2 = a.inv_bc2_sqrt;
    if (a.step_dev) {                       // the count lives in device memory (a launch in a HIP graph keeps its arguments)
        step += *a.step_dev;
        step_size = (float)(a.lr / (1.0 - pow(a.beta1, (double)step)));
        inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)step)));
    }
    P* p = (P*)t.p;
    const G* g = (const G*)t.g;
    float *m32 = (float*)t.m, *v32 = (float*)t.v;
    unsigned char *m8 = (unsigned char*)t.m, *v8 = (unsigned char*)t.v;
    unsigned long long key = 0;
    if constexpr (BITS == 8) key = mix64(a.seed + 0x9E3779B97F4A7C15ULL * ((unsigned long long)step * (1ull << 20) + (t.index & ~AT_VEC)));

    if ((t.index & AT_VEC) && base + AT_WAVE_BLOCKS * AT_BLOCK <= n) {
        // everything is asked for before anything is used: the loads of four blocks are in flight together
        f32x4 pp[AT_WAVE_BLOCKS], gg[AT_WAVE_BLOCKS], mm[AT_WAVE_BLOCKS], vv[AT_WAVE_BLOCKS];
        unsigned mc[AT_WAVE_BLOCKS], vc[AT_WAVE_BLOCKS];
        float ms[AT_WAVE_BLOCKS], vs[AT_WAVE_BLOCKS];
        const long long i0 = base + lane * 4;
#pragma unroll
        for (int b = 0; b < AT_WAVE_BLOCKS; ++b) {
            const long long i = i0 + b * AT_BLOCK;
            pp[b] = load4<P>(p + i);
            gg[b] = load4<G>(g + i);
            if constexpr (BITS == 32) { mm[b] = load4<float>(m32 + i); vv[b] = load4<float>(v32 + i); }
            else {
                mc[b] = *reinterpret_cast<const unsigned*>(m8 + i);
                vc[b] = *reinterpret_cast<const unsigned*>(v8 + i);
                ms[b] = t.ms[blk + b];
                vs[b] = t.vs[blk + b];
            }
        }
#pragma unroll
        for (int b = 0; b < AT_WAVE_BLOCKS; ++b) {
            const long long i = i0 + b * AT_BLOCK;
            adamw_four<BITS>(a, step_size, inv_bc2, key, i, pp[b], gg[b], mm[b], vv[b], mc[b], vc[b], ms[b], vs[b]);
            put4<P>(p + i, pp[b]);
            if constexpr (BITS == 32) { put4<float>(m32 + i, mm[b]); put4<float>(v32 + i, vv[b]); }
            else {
                *reinterpret_cast<unsigned*>(m8 + i) = mc[b];
                *reinterpret_cast<unsigned*>(v8 + i) = vc[b];
                if (lane == 0) { t.ms[blk + b] = ms[b]; t.vs[blk + b] = vs[b]; }
            }
        }
        return;
    }
    // a tensor's end, or one that is not aligned: value by value
    for (int b = 0; b < AT_WAVE_BLOCKS && base + b * AT_BLOCK < n; ++b) {
        const long long i = base + b * AT_BLOCK + lane * 4;
        const int have = i + 4 <= n ? 4 : (i < n ? (int)(n - i) : 0);
        f32x4 pp = {0.f, 0.f, 0.f, 0.f}, gg = pp, mm = pp, vv = pp;
        unsigned mc = 0, vc = 0;
        float ms = 0.f, vs = 0.f;
        for (int e = 0; e < have; ++e) {
            pp[e] = (float)p[i + e];
            gg[e] = (float)g[i + e];
            if constexpr (BITS == 32) { mm[e] = m32[i + e]; vv[e] = v32[i + e]; }
            else { mc |= (unsigned)m8[i + e] << (8 * e); vc |= (unsigned)v8[i + e] << (8 * e); }
        }
        if constexpr (BITS == 8) { ms = t.ms[blk + b]; vs = t.vs[blk + b]; }
        adamw_four<BITS>(a, step_size, inv_bc2, key, i, pp, gg, mm, vv, mc, vc, ms, vs);
        for (int e = 0; e < have; ++e) {
            p[i + e] = (P)pp[e];
            if constexpr (BITS == 32) { m32[i + e] = mm[e]; v32[i + e] = vv[e]; }
            else { m8[i + e] = (unsigned char)(mc >> (8 * e)); v8[i + e] = (unsigned char)(vc >> (8 * e)); }
        }
        if constexpr (BITS == 8)
            if (lane == 0) { t.ms[blk + b] = ms; t.vs[blk + b] = vs; }
    }
}

static size_t size_of(int dt) { return dt == DT_F32 ? 4 : 2; }

template <typename P, typename G>
static void adamw_go(const AdamTable& a, int bits, unsigned blocks, hipStream_t st) {
    if (bits == 32) hipLaunchKernelGGL((adamw_tensors_kernel<P, G, 32>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((adamw_tensors_kernel<P, G, 8>), dim3(blocks), dim3(256), 0, st, a);
}

int adamw_tensors(int count, void* const* p, const void* const* g, void* const* m, void* const* v, float* const* ms, float* const* vs,
                  const long long* n, const int* steps, const int* index, int p_dtype, int g_dtype, int bits, double lr, double beta1,
                  double beta2, double eps, double weight_decay, double grad_scale, unsigned long long seed, const int* step_dev,
                  hipStream_t st) {
    if (count < 0 || (count > 0 && (!p || !g || !m || !v || !n || !steps || !index)) || (bits == 8 && count > 0 && (!ms || !vs))) {
        set_error("adamw_tensors: null list");
        return ICAP_ERR_ARG;
    }
    if ((bits != 8 && bits != 32) || p_dtype < 0 || p_dtype > 2 || (g_dtype != p_dtype && g_dtype != DT_F32)) {
        set_error("adamw_tensors: states of 8 or 32 bits, parameters fp32 / bf16 / fp16, gradients of the same type or fp32");
        return ICAP_ERR_ARG;
    }
    for (int i = 0; i < count; ++i) {       // everything is looked at before anything is launched
        if (n[i] < 0 || (n[i] > 0 && (!p[i] || !g[i] || !m[i] || !v[i] || (bits == 8 && (!ms[i] || !vs[i])))) || index[i] < 0 || index[i] >= (1 << 20) ||
            (!step_dev && steps[i] < 1)) {
            set_error("adamw_tensors: tensor %d: null pointer, size, index (below 2^20) or step (from 1)", i);
            return ICAP_ERR_ARG;
        }
        if (n[i] > (1ll << 40)) { set_error("adamw_tensors: tensor %d is too large", i); return ICAP_ERR_LIMIT; }
    }
    AdamTable a;
    a.decay = (float)(1.0 - lr * weight_decay);
    a.one_minus_b1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2;
    a.one_minus_b2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.grad_scale = (float)grad_scale;
    a.seed = seed;
    a.step_dev = step_dev;
    a.lr = lr; a.beta1 = beta1; a.beta2 = beta2;
    // tensors of one step go together (a parameter that got its first gradient late has a count of its own)
    bool any = false;
    long long above = -(1ll << 40);
    for (;;) {
        long long step = 1ll << 40;
        for (int i = 0; i < count; ++i)
            if (n[i] > 0 && steps[i] > above && steps[i] < step) step = steps[i];
        if (step == 1ll << 40) break;
        above = step;
        a.step = (int)step;
        if (!step_dev) {
            a.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
            a.inv_bc2_sqrt = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
        }
        int i = 0;
        while (i < count) {
            a.count = 0;
            unsigned blocks = 0;
            for (; i < count && a.count < AT_MAX; ++i) {
                if (n[i] == 0 || steps[i] != step) continue;
                const long long need = (n[i] + AT_CHUNK - 1) / AT_CHUNK;
                if (blocks + need > 0x7fffffffLL) break;
                AdamTensor& t = a.t[a.count++];
                t.p = p[i]; t.g = g[i]; t.m = m[i]; t.v = v[i];
                t.ms = bits == 8 ? ms[i] : nullptr;
                t.vs = bits == 8 ? vs[i] : nullptr;
                t.n = n[i];
                t.first = blocks;
                const size_t sp = 4 * size_of(p_dtype), sg = 4 * size_of(g_dtype), ss = bits == 8 ? 4 : 16;
                const bool vec = (uintptr_t)p[i] % sp == 0 && (uintptr_t)g[i] % sg == 0 && (uintptr_t)m[i] % ss == 0 && (uintptr_t)v[i] % ss == 0;
                t.index = (unsigned)index[i] | (vec ? AT_VEC : 0u);
                blocks += (unsigned)need;
            }
            if (!blocks) continue;
            any = true;
            const int key = p_dtype * 3 + g_dtype;
            if (key == DT_F32 * 3 + DT_F32) adamw_go<float, float>(a, bits, blocks, st);
            else if (key == DT_BF16 * 3 + DT_BF16) adamw_go<__bf16, __bf16>(a, bits, blocks, st);
            else if (key == DT_BF16 * 3 + DT_F32) adamw_go<__bf16, float>(a, bits, blocks, st);
            else if (key == DT_F16 * 3 + DT_F16) adamw_go<_Float16, _Float16>(a, bits, blocks, st);
            else adamw_go<_Float16, float>(a, bits, blocks, st);
        }
    }
    return any ? launch_status("adamw_tensors") : ICAP_OK;
}

}  // namespace icap
