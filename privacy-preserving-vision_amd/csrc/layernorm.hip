// Layer norm over the last axis, forward and backward with the weight gradient's reduction (gfx950).
//
//     mean = sum_c x / C,  rstd = 1 / sqrt(sum_c (x - mean)^2 / C + eps),  h = (x - mean) rstd,  y = h w + b
//     dx = rstd (g w - mean_c(g w) - h mean_c(g w h)),  dw = sum_rows g h,  db = sum_rows g
//
// Byte-bound: forward reads x and writes y, backward reads x and g and writes dx, once each.  A row is held in registers by LPR lanes
// (16, a wave, or a workgroup), NV 16-byte vectors each, so the variance is the two-pass one (sum of squared distances from the mean: no
// cancellation for rows far from zero) without reading the row again.  All sums are f32.  Rows may start at any element: the 16-byte
// loads ask for element alignment only (global memory takes them), the last vector of a row is read from where it is whole (elem_types.h).
// Both directions: a fixed grid strides over the rows, the parameters are in registers, the next row is on its way while one is worked on.
// Backward: every lane keeps the weight-gradient sums of its columns in registers, a workgroup leaves one partial row, a second launch adds the partial rows in their order (no atomics:
// the same bits every time).
// Measured (MI355X, bytes read and written once): 165888 x 2048 bf16 forward 266 us = 5.1 TB/s, backward 369 + 4 = 5.5 (638 us a pass; 816 without the next
// row's loads in the backward kernel); f32 of 300 columns and more 4.7-5.7 and 4.9-5.5; 16-bit rows of an odd C, which start off every dword, 3.9-4.6 and
// 2.6-4.3; rows longer than 8192, read again for each pass, 2.4-3.4 and 1.6-2.5.  6656 x 512 bf16: 6 + 8 + 4 us, less than the host takes to ask for them.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include "ppv_common.h"
#include "ppv_hip.h"
#include "elem_types.h"

namespace ppv {

// sum over the LPR lanes of a row's group, the same value (same order of additions) in each of them
template <int LPR> __device__ __forceinline__ float group_sum(float v, float* lds) {
    v = row16_sum_f(v);
    if constexpr (LPR >= 64) v = wave_sum_of_rows(v);
    if constexpr (LPR > 64) {
        constexpr int NW = LPR / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        const int w0 = threadIdx.x / LPR * NW;
        v = lds[w0];
#pragma unroll
        for (int i = 1; i < NW; ++i) v += lds[w0 + i];
        __syncthreads();                                       // the next sum writes the same words
    }
    return v;
}

template <class T, int LPR, int NV, int NT>
__global__ __launch_bounds__(NT) void layernorm_fwd_kernel(const T* __restrict__ x, long ldx, const void* __restrict__ w, const void* __restrict__ b,
                                                           int wdtype, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                           long rows, int C, float eps) {
    constexpr int V = 16 / sizeof(T), RPW = NT / LPR;
    __shared__ float lds[LPR > 64 ? NT / 64 : 1];
    const int l = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const float inv_c = 1.f / (float)C;
    const long step = (long)gridDim.x * RPW, turns = (rows + step - 1) / step, row0 = (long)blockIdx.x * RPW + grp;
    u32x4 raw[NV];
    auto fetch = [&](long row) {
        const T* xr = x + (row < rows ? row : 0) * ldx;
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = load_row_vec<T>(xr, (i * LPR + l) * V, C);
    };
    fetch(row0);
    float wv[NV][V], bv[NV][V];                                // once for all rows of this slot
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        load_param<V>(w, wdtype, (i * LPR + l) * V, C, 1.f, wv[i]);
        load_param<V>(b, wdtype, (i * LPR + l) * V, C, 0.f, bv[i]);
    }
    for (long t = 0; t < turns; ++t) {                         // (a slot without a row keeps running: the sums below cross lanes)
        const long row = t * step + row0;
        float v[NV][V];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * LPR + l) * V;
            if ((i + 1) * LPR * V > C && C >= V) raw[i] = drop_front<T>(raw[i], c - min(c, C - V));
            unpack_vec<T>(raw[i], v[i]);
        }
        if (t + 1 < turns) fetch(row + step);                  // the next row comes while this one is worked on
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[i][e];
        const float mean = group_sum<LPR>(s, lds) * inv_c;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int left = C - (i * LPR + l) * V;
            const bool end = (i + 1) * LPR * V > C;            // (the same for all lanes: the other vectors are whole)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] -= mean;
                if (end && e >= left) v[i][e] = 0.f;
                q = __builtin_fmaf(v[i][e], v[i][e], q);
            }
        }
        const float rstd = 1.f / __builtin_sqrtf(group_sum<LPR>(q, lds) * inv_c + eps);
        if (row >= rows) continue;
        T* yr = y + row * (long)C;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * LPR + l) * V;
            if (c >= C) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = __builtin_fmaf(v[i][e] * rstd, wv[i][e], bv[i][e]);
            store_vec<T, V>(yr + c, C - c, o);
        }
        if (mean_out && l == 0) { mean_out[row] = mean; rstd_out[row] = rstd; }
    }
}

// One workgroup for each of n rows (or 16 columns): a launch counts its work items in 32 bits along an axis, so those beyond 2^16 go along y.
static inline dim3 one_each(long n) { return dim3((unsigned)(n < 65536 ? n : 65536), (unsigned)((n + 65535) / 65536)); }
__device__ __forceinline__ long which_one() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }

// rows longer than the registers hold: three passes over the row (the second and third come out of the L2)
template <class T>
__global__ __launch_bounds__(256) void layernorm_fwd_long_kernel(const T* __restrict__ x, long ldx, const void* __restrict__ w, const void* __restrict__ b,
                                                                 int wdtype, T* __restrict__ y, float* __restrict__ mean_out,
                                                                 float* __restrict__ rstd_out, long rows, int C, float eps) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float lds[4];
    const long row = which_one();
    if (row >= rows) return;
    const T* xr = x + row * ldx;
    float v[V];
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x * V; c < C; c += 256 * V) {
        load_row<T, V>(xr, c, C, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s += v[e];
    }
    const float mean = group_sum<256>(s, lds) / (float)C;
    for (int c = threadIdx.x * V; c < C; c += 256 * V) {
        load_row<T, V>(xr, c, C, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = e < C - c ? v[e] - mean : 0.f;
            q = __builtin_fmaf(d, d, q);
        }
    }
    const float rstd = 1.f / __builtin_sqrtf(group_sum<256>(q, lds) / (float)C + eps);
    T* yr = y + row * (long)C;
    for (int c = threadIdx.x * V; c < C; c += 256 * V) {
        float wv[V], bv[V];
        load_row<T, V>(xr, c, C, v);
        load_param<V>(w, wdtype, c, C, 1.f, wv);
        load_param<V>(b, wdtype, c, C, 0.f, bv);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = __builtin_fmaf((v[e] - mean) * rstd, wv[e], bv[e]);
        store_vec<T, V>(yr + c, C - c, v);
    }
    if (mean_out && threadIdx.x == 0) { mean_out[row] = mean; rstd_out[row] = rstd; }
}

// two sums at once over the LPR lanes of a row's group
template <int LPR> __device__ __forceinline__ void group_sum2(float& a, float& b, float (*lds)[2]) {
    a = row16_sum_f(a);
    b = row16_sum_f(b);
    if constexpr (LPR >= 64) { a = wave_sum_of_rows(a); b = wave_sum_of_rows(b); }
    if constexpr (LPR > 64) {
        constexpr int NW = LPR / 64;
        if ((threadIdx.x & 63) == 0) { lds[threadIdx.x >> 6][0] = a; lds[threadIdx.x >> 6][1] = b; }
        __syncthreads();
        const int w0 = threadIdx.x / LPR * NW;
        a = lds[w0][0];
        b = lds[w0][1];
#pragma unroll
        for (int i = 1; i < NW; ++i) { a += lds[w0 + i][0]; b += lds[w0 + i][1]; }
        __syncthreads();
    }
}

template <class T, int LPR, int NV, int NT>
__global__ __launch_bounds__(NT, 2) void layernorm_bwd_kernel(const T* __restrict__ g, long ldg, const T* __restrict__ x, long ldx,
                                                              const void* __restrict__ w, int wdtype, const float* __restrict__ mean_in,
                                                              const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part,
                                                              long rows, int C) {
    constexpr int V = 16 / sizeof(T), RPW = NT / LPR;
    extern __shared__ float smem[];                            // LPR < NT: the waves' (row slots') sums, [C] each
    __shared__ float lds[LPR > 64 ? NT / 64 : 1][2];
    const int l = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const float inv_c = 1.f / (float)C;
    const long step = (long)gridDim.x * RPW, turns = (rows + step - 1) / step, row0 = (long)blockIdx.x * RPW + grp;
    u32x4 gr[NV], xr[NV];
    float mean, rstd;
    auto fetch = [&](long row) {
        const bool live = row < rows;
        const long at = live ? row : 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * LPR + l) * V;
            gr[i] = load_row_vec<T>(g + at * ldg, c, C);
            xr[i] = load_row_vec<T>(x + at * ldx, c, C);
        }
        mean = mean_in[at];
        rstd = rstd_in[at];
    };
    fetch(row0);
    float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * LPR + l) * V;
        load_param<V>(w, wdtype, c, C, 1.f, wv[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) aw[i][e] = ab[i][e] = 0.f;
    }
    for (long t = 0; t < turns; ++t) {                         // the same number of turns for every lane: the sums cross lanes and waves
        const long row = t * step + row0;
        const bool live = row < rows;
        float gv[NV][V], hv[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * LPR + l) * V;
            if ((i + 1) * LPR * V > C && C >= V) {
                gr[i] = drop_front<T>(gr[i], c - min(c, C - V));
                xr[i] = drop_front<T>(xr[i], c - min(c, C - V));
            }
            if (!live) gr[i] = (u32x4){0, 0, 0, 0};            // (this slot's last turn may have no row)
            unpack_vec<T>(gr[i], gv[i]);
            unpack_vec<T>(xr[i], hv[i]);
        }
        const float mu = mean, rs = rstd;
        if (t + 1 < turns) fetch(row + step);                  // the next row comes while this one is worked on
        __builtin_amdgcn_sched_barrier(0);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int left = C - (i * LPR + l) * V;
            const bool end = (i + 1) * LPR * V > C;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float h = (hv[i][e] - mu) * rs, gw = gv[i][e] * wv[i][e];                              // (g is zero behind the row)
                if (end && e >= left) h = gw = 0.f;
                aw[i][e] = __builtin_fmaf(gv[i][e], h, aw[i][e]);
                ab[i][e] += gv[i][e];
                s1 += gw;
                s2 = __builtin_fmaf(gw, h, s2);
                hv[i][e] = h;
                gv[i][e] = gw;
            }
        }
        group_sum2<LPR>(s1, s2, lds);
        s1 *= inv_c;
        s2 *= inv_c;
        if (!live) continue;
        T* dr = dx + row * (long)C;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * LPR + l) * V;
            if (c >= C) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = rs * (gv[i][e] - s1 - hv[i][e] * s2);
            store_vec<T, V>(dr + c, C - c, o);
        }
    }
    if (!part) return;
    float* pw = part + (long)blockIdx.x * 2 * C;
    if constexpr (LPR < NT) {                                  // several rows at a time in this workgroup: their sums meet in LDS, added in order
        if constexpr (LPR < 64) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) { aw[i][e] = wave_sum_of_rows(aw[i][e]); ab[i][e] = wave_sum_of_rows(ab[i][e]); }
        }
        constexpr int PARTS = LPR <= 64 ? NT / 64 : RPW;
        const int part_of = LPR <= 64 ? threadIdx.x >> 6 : grp;
        auto meet = [&](float (&v)[NV][V], float* out) {
            if (LPR >= 64 || (threadIdx.x & 63) < LPR)
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int c = (i * LPR + l) * V + e;
                        if (c < C) smem[part_of * C + c] = v[i][e];
                    }
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += NT) {
                float s = smem[c];
#pragma unroll
                for (int k = 1; k < PARTS; ++k) s += smem[k * C + c];
                out[c] = s;
            }
        };
        meet(aw, pw);
        __syncthreads();
        meet(ab, pw + C);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = (i * LPR + l) * V + e;
                if (c < C) { pw[c] = aw[i][e]; pw[C + c] = ab[i][e]; }
            }
    }
}

template <class T>
__global__ __launch_bounds__(256) void layernorm_bwd_long_kernel(const T* __restrict__ g, long ldg, const T* __restrict__ x, long ldx,
                                                                 const void* __restrict__ w, int wdtype, const float* __restrict__ mean_in,
                                                                 const float* __restrict__ rstd_in, T* __restrict__ dx, long rows, int C) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float lds[4];
    const long row = which_one();
    if (row >= rows) return;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s1 = 0.f, s2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
        for (int c = threadIdx.x * V; c < C; c += 256 * V) {
            float gv[V], xv[V], wv[V];
            load_row<T, V>(g + row * ldg, c, C, gv);
            load_row<T, V>(x + row * ldx, c, C, xv);
            load_param<V>(w, wdtype, c, C, 1.f, wv);
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float h = e < C - c ? (xv[e] - mean) * rstd : 0.f, gw = gv[e] * wv[e];
                if (pass == 0) { s1 += gw; s2 = __builtin_fmaf(gw, h, s2); }
                o[e] = rstd * (gw - s1 - h * s2);
            }
            if (pass == 1) store_vec<T, V>(dx + row * (long)C + c, C - c, o);
        }
        if (pass == 0) {
            s1 = group_sum<256>(s1, lds) / (float)C;
            s2 = group_sum<256>(s2, lds) / (float)C;
        }
    }
}

// weight-gradient partials of the long rows: a thread owns a column, a workgroup row of the grid strides over the rows
template <class T>
__global__ __launch_bounds__(256) void layernorm_wgrad_long_kernel(const T* __restrict__ g, long ldg, const T* __restrict__ x, long ldx,
                                                                   const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                   float* __restrict__ part, long rows, int C) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    float aw = 0.f, ab = 0.f;
    for (long r = blockIdx.y; r < rows; r += gridDim.y) {
        const float gv = to_f32(g[r * ldg + c]);
        aw = __builtin_fmaf(gv, (to_f32(x[r * ldx + c]) - mean_in[r]) * rstd_in[r], aw);
        ab += gv;
    }
    part[(long)blockIdx.y * 2 * C + c] = aw;
    part[(long)blockIdx.y * 2 * C + C + c] = ab;
}

// part [G][2][C] -> dw, db: 16 columns x 16 slices of the partial rows per workgroup, the slices added in order
__global__ __launch_bounds__(256) void layernorm_wgrad_reduce_kernel(const float* __restrict__ part, int G, int C, void* __restrict__ dw,
                                                                     void* __restrict__ db, int wdtype) {
    __shared__ float s[16][17];
    const int j = threadIdx.x & 15, k = threadIdx.x >> 4;
    const long c = which_one() * 16 + j;                       // over the 2 C columns of a partial row
    float a = 0.f;
    if (c < 2L * C) {
#pragma unroll 8
        for (int r = k; r < G; r += 16) a += part[(long)r * 2 * C + c];
    }
    s[k][j] = a;
    __syncthreads();
    if (k == 0 && c < 2L * C) {
#pragma unroll
        for (int i = 1; i < 16; ++i) a += s[i][j];
        void* out = c < C ? dw : db;
        if (out) store_param(out, wdtype, c < C ? c : c - C, a);
    }
}

// workgroups of the backward pass: two for each CU (165888 rows of 2048 bf16: 512 and 256 take 620 us with the forward pass, 768 650, 1024 690,
// 2048 710: more streams at once are worse for the memory), at least four rows for each row slot, so that the partial rows stay few
static int layernorm_bwd_groups(long rows, int C, int rpw) {
    const long by_rows = (rows + 4L * rpw - 1) / (4L * rpw);
    const long most = C > 8192 ? 64 : 512;
    return (int)(by_rows < 1 ? 1 : by_rows > most ? most : by_rows);
}
// lanes per row: at most 16 elements a lane (two gradient sums, a weight and two operands each; with 32 the next row's
// loads no longer fit beside them), 0: longer than the registers hold
static int layernorm_lpr(int C, int dtype) {
    const int v = dtype == 0 ? 4 : 8, nvec = (C + v - 1) / v, most = 16 / v;
    return nvec <= 16 ? 16 : nvec <= 64 * most ? 64 : nvec <= 128 * most ? 128 : nvec <= 256 * most ? 256 : nvec <= 512 * most ? 512 : 0;
}
static int layernorm_groups_of(long rows, int C, int dtype) {
    const int lpr = layernorm_lpr(C, dtype);
    return layernorm_bwd_groups(rows, C, lpr == 0 || lpr >= 256 ? 1 : 256 / lpr);
}

constexpr long FWD_GROUPS = 1024;
template <class T>
static int layernorm_fwd_t(const T* x, long ldx, const void* w, const void* b, int wdtype, T* y, float* mean, float* rstd, long rows, int C,
                           float eps, hipStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const int nvec = (C + V - 1) / V, lpr = layernorm_lpr(C, sizeof(T) == 4 ? 0 : 1);
    // four workgroups of 256 threads for each CU, each with as many rows as that takes (2048 and more are no faster)
    auto grid = [&](int rpw, long most) { const long n = (rows + rpw - 1) / rpw; return (unsigned)(n < most ? n : most); };
#define LN_FWD(LPR, NV, NT) \
    layernorm_fwd_kernel<T, LPR, NV, NT><<<grid(NT / LPR, NT == 512 ? 1024 : FWD_GROUPS), NT, 0, stream>>>(x, ldx, w, b, wdtype, y, mean, rstd, rows, C, eps)
    if (lpr == 16) LN_FWD(16, 1, 256);
    else if (lpr == 64 && nvec <= 64) LN_FWD(64, 1, 256);
    else if (lpr == 64 && nvec <= 128) LN_FWD(64, 2, 256);
    else if (lpr == 64) LN_FWD(64, 16 / V, 256);               // (f32: 4 vectors; the 16-bit types end at 2)
    else if (lpr == 128) LN_FWD(128, 16 / V, 256);
    else if (lpr == 256) LN_FWD(256, 16 / V, 256);
    else if (lpr == 512) LN_FWD(512, 16 / V, 512);
    else if (rows > 0x7fffffffL) return PPV_ERR_BAD_SIZE;
    else layernorm_fwd_long_kernel<T><<<one_each(rows), 256, 0, stream>>>(x, ldx, w, b, wdtype, y, mean, rstd, rows, C, eps);
#undef LN_FWD
    return ppv_last_error();
}

template <class T>
static int layernorm_bwd_t(const T* g, long ldg, const T* x, long ldx, const void* w, int wdtype, const float* mean, const float* rstd, T* dx,
                           void* dw, void* db, float* part, long rows, int C, int dtype, hipStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const int nvec = (C + V - 1) / V, lpr = layernorm_lpr(C, dtype), G = layernorm_groups_of(rows, C, dtype);
    if (!dw && !db) part = nullptr;
#define LN_BWD(LPR, NV, NT)                                                                                                              \
    layernorm_bwd_kernel<T, LPR, NV, NT><<<G, NT, (LPR >= NT ? 0 : LPR <= 64 ? NT / 64 : NT / LPR) * C * sizeof(float), stream>>>(        \
        g, ldg, x, ldx, w, wdtype, mean, rstd, dx, part, rows, C)
    if (lpr == 16) LN_BWD(16, 1, 256);
    else if (lpr == 64 && nvec <= 64) LN_BWD(64, 1, 256);
    else if (lpr == 64 && nvec <= 128) LN_BWD(64, 2, 256);
    else if (lpr == 64) LN_BWD(64, 16 / V, 256);               // (f32: 4 vectors; the 16-bit types end at 2)
    else if (lpr == 128) LN_BWD(128, 16 / V, 256);
    else if (lpr == 256) LN_BWD(256, 16 / V, 256);
    else if (lpr == 512) LN_BWD(512, 16 / V, 512);
    else {
        if (rows > 0x7fffffffL) return PPV_ERR_BAD_SIZE;
        layernorm_bwd_long_kernel<T><<<one_each(rows), 256, 0, stream>>>(g, ldg, x, ldx, w, wdtype, mean, rstd, dx, rows, C);
        if (part) layernorm_wgrad_long_kernel<T><<<dim3((C + 255) / 256, G), 256, 0, stream>>>(g, ldg, x, ldx, mean, rstd, part, rows, C);
    }
#undef LN_BWD
    if (part) layernorm_wgrad_reduce_kernel<<<one_each((2L * C + 15) / 16), 256, 0, stream>>>(part, G, C, dw, db, wdtype);
    return ppv_last_error();
}

}  // namespace ppv

using namespace ppv;

extern "C" {

int ppv_layernorm_fwd(const void* x, long ldx, const void* w, const void* b, void* y, float* mean, float* rstd, long rows, int C, int dtype,
                      int wdtype, float eps, hipStream_t stream) {
    if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return PPV_ERR_NULL;
    if (rows < 1 || C < 1 || C > (1 << 30) || ldx < 0 || dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2) return PPV_ERR_BAD_SIZE;
    if (dtype == 0) return layernorm_fwd_t((const float*)x, ldx, w, b, wdtype, (float*)y, mean, rstd, rows, C, eps, stream);
    if (dtype == 1) return layernorm_fwd_t((const bf16s*)x, ldx, w, b, wdtype, (bf16s*)y, mean, rstd, rows, C, eps, stream);
    return layernorm_fwd_t((const f16s*)x, ldx, w, b, wdtype, (f16s*)y, mean, rstd, rows, C, eps, stream);
}

size_t ppv_layernorm_bwd_workspace_bytes(long rows, int C, int dtype) {
    if (rows < 1 || C < 1 || C > (1 << 30) || dtype < 0 || dtype > 2) return 0;
    return (size_t)layernorm_groups_of(rows, C, dtype) * 2 * (size_t)C * sizeof(float);
}

int ppv_layernorm_bwd(const void* g, long ldg, const void* x, long ldx, const void* w, const float* mean, const float* rstd, void* dx, void* dw,
                      void* db, void* workspace, long rows, int C, int dtype, int wdtype, hipStream_t stream) {
    if (!g || !x || !mean || !rstd || !dx || ((dw || db) && !workspace)) return PPV_ERR_NULL;
    if (rows < 1 || C < 1 || C > (1 << 30) || ldx < 0 || ldg < 0 || dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2) return PPV_ERR_BAD_SIZE;
    float* part = (float*)workspace;
    if (dtype == 0)
        return layernorm_bwd_t((const float*)g, ldg, (const float*)x, ldx, w, wdtype, mean, rstd, (float*)dx, dw, db, part, rows, C, dtype, stream);
    if (dtype == 1)
        return layernorm_bwd_t((const bf16s*)g, ldg, (const bf16s*)x, ldx, w, wdtype, mean, rstd, (bf16s*)dx, dw, db, part, rows, C, dtype, stream);
    return layernorm_bwd_t((const f16s*)g, ldg, (const f16s*)x, ldx, w, wdtype, mean, rstd, (f16s*)dx, dw, db, part, rows, C, dtype, stream);
}

}  // extern "C"
