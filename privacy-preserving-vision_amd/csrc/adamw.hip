// AdamW step of a whole parameter list in one launch, moments in 32 or in 8 bits (gfx950).
//
//     m = m + (1 - b1)(g - m);   v = b2 v + (1 - b2) g^2;   r = sqrt(v)
//     p = (1 - lr wd) p - lr / (1 - b1^t) * m / (r / sqrt(1 - b2^t) + eps)
//
// Byte-bound: 28 bytes per parameter with 32-bit moments (p, g, m, v read; p, m, v written), 16 with 8-bit moments.  As in optim.hip every
// 4096-element chunk of every tensor is a workgroup of the one launch, all its loads requested before the first store.
//
// 8-bit moments: m and r (the ROOT of v: half the range in powers of two, and the quantity the update divides by) as OCP e4m3 values in blocks
// of 256 consecutive elements with one f32 scale each.
//  * Scales are powers of two, 2^(floor(log2 max) - 7), so that a value that does not change keeps its code when the block's maximum
//    moves: codes only see rounding where the moment itself moves.
//  * Rounding is stochastic (up with the probability of the nearness of the upper neighbour; 16 random bits per value, a 32-bit integer
//    hash of seed, step, tensor and element, so a run repeats bit for bit).  With beta2 = 0.999 a second moment moves by ~1e-3 per step,
//    an e4m3 step is 6-12 %: rounded to nearest it would stay where it is for ever.
//  * A root that is not zero never becomes zero: m / eps would be a jump.  Values that are not finite become NaN codes and stay out of
//    the block's maximum.
// All arithmetic is f32 with every operation rounded by itself: the codes are a function of the inputs that can be stated, and recomputed
// elsewhere, exactly.  (The Makefile compiles this file with -ffp-contract=off; under =fast the pragma of that name does not hold.)
// Measured (MI355X): 20.5 M elements, 32 bits: 94 us = 6.1 TB/s step after step on one list, 114 us = 5.0 on lists in turn (nothing of them left in the
// caches); 63 M elements in 333 tensors, 8 bits: 196 us = 5.2 TB/s.
#include <hip/hip_runtime.h>
#include <cmath>
#include "ppv_common.h"
#include "ppv_hip.h"
#include "elem_types.h"

namespace ppv {

// ms != null: 8-bit moments (m, v: e4m3 codes of m and r; ms, vs: a scale per 256 elements); else m, v are f32.  64 bytes.
struct AdamWDesc { float* p; const float* g; void* m; void* v; float* ms; float* vs; long numel; int blk0; unsigned stream; };
constexpr int AW_NT = 256, AW_IT = 4, AW_CHUNK = AW_NT * AW_IT * 4;

struct AdamWArgs { float decay, rate, undo, b1c, b2, b2c, eps; unsigned key; };

__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, float& root, const AdamWArgs& a) {
    m = m + (g - m) * a.b1c;
    v = v * a.b2 + (g * a.b2c) * g;
    root = __builtin_sqrtf(v);
    p = p * a.decay - (m / (root * a.undo + a.eps)) * a.rate;
}

// the tensors' addresses come out of a table: named global here, or their loads would be flat ones
#define AW_GLOBAL __attribute__((address_space(1)))
typedef float F4 __attribute__((ext_vector_type(4)));
typedef AW_GLOBAL float GF;
typedef AW_GLOBAL unsigned char GB;
typedef float F4A __attribute__((ext_vector_type(4), aligned(4)));             // (any element may start a tensor)
typedef unsigned W1A __attribute__((aligned(1)));

// The mixer is the one published in C. Wellons, "Prospecting for Hash Functions" (2018): multipliers 0x7FEB352D and 0x846CA68B, shifts 16, 15, 16.
// Element, step and tensor go in spread by the usual hash primes 0x9E3779B1, 0x85EBCA77 and 0xC2B2AE3D.
__device__ __forceinline__ unsigned adamw_hash(unsigned i, unsigned key) {
    unsigned h = i * 0x9E3779B1u + key;
    h = (h ^ (h >> 16)) * 0x7FEB352Du;
    h = (h ^ (h >> 15)) * 0x846CA68Bu;
    return h ^ (h >> 16);
}
// e4m3 code of a = |x| / scale < 256 with 16 bits of dither; `keep`: not down to zero
__device__ __forceinline__ unsigned e4m3_stochastic(float a, unsigned dither, bool keep) {
    const unsigned up = dither * 16 + 8;
    if (!(a < __builtin_inff())) return 0x7Fu;
    const unsigned normal = ((__builtin_bit_cast(unsigned, a) + up) >> 20) - (120u << 3);
    const unsigned small = (unsigned)__builtin_floorf(a * 512.f + (float)up * 0x1p-20f);
    const unsigned code = a >= 0x1p-6f ? normal : small;
    return code == 0 && keep && a > 0.f ? 1u : code;
}
__device__ __forceinline__ unsigned umax_row(unsigned v) {
    auto step = [](unsigned x, unsigned y) { return x > y ? x : y; };
    v = step(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));
    v = step(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));
    v = step(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));
    v = step(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = step((unsigned)a[0], (unsigned)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return step((unsigned)b[0], (unsigned)b[1]);
}
// exponent field (biased) that a block's scale is made from: floor(log2 max) kept where 2^(e - 7) and 2^(7 - e) are both normal numbers
__device__ __forceinline__ unsigned block_exp(const float (&x)[4], unsigned left) {
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned b = __builtin_bit_cast(unsigned, x[e]) & 0x7fffffffu;
        if (b < 0x7f800000u && e < (int)left && b > top) top = b;
    }
    const unsigned f = umax_row(top) >> 23;
    return f < 9 ? 9 : f;
}

__global__ __launch_bounds__(AW_NT) void adamw_multi_kernel(const AdamWDesc* __restrict__ desc, int ndesc, AdamWArgs a) {
    int lo = 0, hi = ndesc - 1;                                 // the tensor that owns this block
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (desc[mid].blk0 <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const AdamWDesc d = desc[lo];
    const long base = (long)((int)blockIdx.x - d.blk0) * AW_CHUNK;
    F4 p[AW_IT], g[AW_IT];
    const bool whole = base + AW_CHUNK <= d.numel;
    auto fetch = [&](const void* src_, int it) {
        const long i = base + (long)(it * AW_NT + threadIdx.x) * 4;
        const GF* src = (const GF*)(const float*)src_;
        F4 r;
        if (whole) r = *(const AW_GLOBAL F4A*)(src + i);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = i + e < d.numel ? src[i + e] : 0.f;
        return r;
    };
    auto put = [&](void* dst_, int it, const F4 v) {
        const long i = base + (long)(it * AW_NT + threadIdx.x) * 4;
        GF* dst = (GF*)(float*)dst_;
        if (whole) *(AW_GLOBAL F4A*)(dst + i) = v;
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < d.numel) dst[i + e] = v[e];
    };
    if (d.ms == nullptr) {
        F4 m[AW_IT], v[AW_IT];
#pragma unroll
        for (int it = 0; it < AW_IT; ++it) {
            p[it] = fetch(d.p, it);
            g[it] = fetch(d.g, it);
            m[it] = fetch(d.m, it);
            v[it] = fetch(d.v, it);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int it = 0; it < AW_IT; ++it) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float root, pe = p[it][e], me = m[it][e], ve = v[it][e];
                adamw_one(pe, g[it][e], me, ve, root, a);
                p[it][e] = pe; m[it][e] = me; v[it][e] = ve;
            }
            put(d.p, it, p[it]);
            put(d.m, it, m[it]);
            put(d.v, it, v[it]);
        }
        return;
    }
    // 8-bit moments: iteration `it` of a wave is one block of 256 elements, four consecutive ones per lane
    unsigned mw[AW_IT], vw[AW_IT];
    float msc[AW_IT], vsc[AW_IT];
    const long blk = base / 256 + (threadIdx.x >> 6);
    auto fetch8 = [&](const void* src, int it) {
        const long i = base + (long)(it * AW_NT + threadIdx.x) * 4;
        const GB* s = (const GB*)(const unsigned char*)src + i;
        unsigned w = 0;
        if (whole) w = *(const AW_GLOBAL W1A*)s;
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < d.numel) w |= (unsigned)s[e] << (8 * e);
        return w;
    };
    auto put8 = [&](void* dst, int it, unsigned w) {
        const long i = base + (long)(it * AW_NT + threadIdx.x) * 4;
        GB* s = (GB*)(unsigned char*)dst + i;
        if (whole) *(AW_GLOBAL W1A*)s = w;
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < d.numel) s[e] = (unsigned char)(w >> (8 * e));
    };
#pragma unroll
    for (int it = 0; it < AW_IT; ++it) {
        const bool some = (blk + it * 4) * 256 < d.numel;
        p[it] = fetch(d.p, it);
        g[it] = fetch(d.g, it);
        mw[it] = fetch8(d.m, it);
        vw[it] = fetch8(d.v, it);
        msc[it] = some ? ((const GF*)d.ms)[blk + it * 4] : 0.f;
        vsc[it] = some ? ((const GF*)d.vs)[blk + it * 4] : 0.f;
    }
    __builtin_amdgcn_sched_barrier(0);
    const unsigned key = a.key + d.stream * 0xC2B2AE3Du;
#pragma unroll
    for (int it = 0; it < AW_IT; ++it) {
        const long i = base + (long)(it * AW_NT + threadIdx.x) * 4;
        const unsigned left = i >= d.numel ? 0u : d.numel - i < 4 ? (unsigned)(d.numel - i) : 4u;
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mw[it], false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mw[it], true);
        const f32x2 r01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vw[it], false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vw[it], true);
        float m[4] = {m01.x * msc[it], m01.y * msc[it], m23.x * msc[it], m23.y * msc[it]};
        float r[4] = {r01.x * vsc[it], r01.y * vsc[it], r23.x * vsc[it], r23.y * vsc[it]};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = r[e] * r[e], pe = p[it][e];
            adamw_one(pe, g[it][e], m[e], v, r[e], a);
            p[it][e] = pe;
        }
        const unsigned me = block_exp(m, left), re = block_exp(r, left);
        const float mi = __builtin_bit_cast(float, (261u - me) << 23), ri = __builtin_bit_cast(float, (261u - re) << 23);   // 2^(7 - e)
        unsigned mc = 0, rc = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned h = adamw_hash((unsigned)(i + e), key);
            const unsigned sign = __builtin_bit_cast(unsigned, m[e]) >> 31;
            mc |= (e4m3_stochastic(__builtin_fabsf(m[e]) * mi, h & 0xffffu, false) | sign << 7) << (8 * e);
            rc |= e4m3_stochastic(r[e] * ri, h >> 16, true) << (8 * e);
        }
        put(d.p, it, p[it]);
        put8(d.m, it, mc);
        put8(d.v, it, rc);
        if ((threadIdx.x & 63) == 0 && left) {
            ((GF*)d.ms)[blk + it * 4] = __builtin_bit_cast(float, (me - 7) << 23);
            ((GF*)d.vs)[blk + it * 4] = __builtin_bit_cast(float, (re - 7) << 23);
        }
    }
}

}  // namespace ppv

using namespace ppv;

extern "C" {

int ppv_adamw_multi(const void* desc, int ndesc, int total_blocks, double lr, double beta1, double beta2, double eps, double weight_decay,
                    double step, unsigned seed, hipStream_t stream) {
    if (!desc) return PPV_ERR_NULL;
    if (ndesc < 1 || total_blocks < 1 || !(step >= 1.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return PPV_ERR_BAD_SIZE;
    AdamWArgs a;
    a.decay = (float)(1.0 - lr * weight_decay);
    a.rate = (float)(lr / (1.0 - std::pow(beta1, step)));
    a.undo = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, step)));
    a.b1c = (float)(1.0 - beta1);
    a.b2 = (float)beta2;
    a.b2c = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.key = seed * 0x9E3779B1u + (unsigned)(unsigned long long)step * 0x85EBCA77u;
    adamw_multi_kernel<<<total_blocks, AW_NT, 0, stream>>>((const AdamWDesc*)desc, ndesc, a);
    return ppv_last_error();
}

}  // extern "C"
