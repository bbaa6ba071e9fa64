// Element types of the kernels that take f32, bf16 or f16 tensors (layernorm.hip, attention*.hip): conversions, 16-byte vectors at element
// alignment with a checked end, sums across lanes.
#pragma once
#include <hip/hip_runtime.h>

namespace ppv {

struct bf16s { unsigned short u; };
struct f16s { unsigned short u; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16s v) { return __builtin_bit_cast(float, (unsigned)v.u << 16); }
__device__ __forceinline__ float to_f32(f16s v) { return (float)__builtin_bit_cast(_Float16, v.u); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16s from_f32<bf16s>(float v) { return {__builtin_bit_cast(unsigned short, (__bf16)v)}; }
template <> __device__ __forceinline__ f16s from_f32<f16s>(float v) { return {__builtin_bit_cast(unsigned short, (_Float16)v)}; }

// 16 bytes at the alignment of one element: ONE load / store (a struct of elements is taken apart by the compiler)
template <class T> struct Raw16;
template <> struct Raw16<float> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Raw16<bf16s> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Raw16<f16s> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <class T> __device__ __forceinline__ void unpack_vec(const u32x4 r, float (&o)[16 / sizeof(T)]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) o[i] = __builtin_bit_cast(float, (unsigned)r[i]);
        else {
            o[2 * i] = to_f32(T{(unsigned short)(r[i] & 0xffffu)});
            o[2 * i + 1] = to_f32(T{(unsigned short)(r[i] >> 16)});
        }
    }
}
template <class T> __device__ __forceinline__ u32x4 pack_vec(const float (&v)[16 / sizeof(T)]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) r[i] = __builtin_bit_cast(unsigned, v[i]);
        else {
            typedef float f32x2_t __attribute__((ext_vector_type(2)));
            const f32x2_t two = {v[2 * i], v[2 * i + 1]};
            if constexpr (__is_same(T, bf16s)) {
                typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
                r[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(two, bf16x2_t));
            } else {
                typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
                r[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(two, f16x2_t));
            }
        }
    }
    return r;
}

// Vectors of a row of C elements without conditions: column c of the row is asked for at min(c, C - V), so the row's last vector, which may not
// be whole, lies inside the row and every lane loads; `drop` = c - min(c, C - V) elements are then taken off its front, with zeros behind
// (V or more: all zeros).  Loads under a condition are waited for one by one.  C < V: element by element.
template <class T> __device__ __forceinline__ u32x4 load_row_vec(const T* row, int c, int C) {
    constexpr int V = 16 / sizeof(T);
    if (C >= V) return *reinterpret_cast<const typename Raw16<T>::type*>(row + min(c, C - V));
    u32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (c + e < C) {
            if constexpr (sizeof(T) == 4) r[e] = *reinterpret_cast<const unsigned*>(row + c + e);
            else r[e / 2] |= (unsigned)row[c + e].u << (16 * (e & 1));
        }
    return r;
}
template <class T> __device__ __forceinline__ u32x4 drop_front(u32x4 r, int drop) {
    constexpr int V = 16 / sizeof(T);
    if (sizeof(T) == 2 && (drop & 1)) r = (u32x4){r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
    if (drop & (V / 4)) r = (u32x4){r[1], r[2], r[3], 0};
    if (drop & (V / 2)) r = (u32x4){r[2], r[3], 0, 0};
    return drop >= V ? (u32x4){0, 0, 0, 0} : r;
}
template <class T, int V> __device__ __forceinline__ void load_row(const T* row, int c, int C, float (&o)[V]) {
    u32x4 r = load_row_vec<T>(row, c, C);
    if (C >= V && __builtin_amdgcn_ballot_w64(c > C - V)) r = drop_front<T>(r, c - min(c, C - V));
    unpack_vec<T>(r, o);
}
template <class T, int V> __device__ __forceinline__ void store_vec(T* p, int left, const float (&v)[V]) {
    static_assert(V * sizeof(T) == 16, "one 16-byte vector");
    if (left >= V) *reinterpret_cast<typename Raw16<T>::type*>(p) = pack_vec<T>(v);
    else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < left) p[e] = from_f32<T>(v[e]);
    }
}
// V elements at column c of a parameter row of run-time type (0 f32, 1 bf16, 2 f16), as load_row_vec; `fill` where there is none, anything behind C
template <class T, int V> __device__ __forceinline__ void load_param_t(const T* p, int c, int C, float (&o)[V]) {
    constexpr int W = 16 / sizeof(T);                          // V is W, 2 W (f32 beside 16-bit rows) or W / 2 (16-bit beside f32 rows)
    if (C >= V) {
        const int at = min(c, C - V), drop = c - at;
        if constexpr (V >= W) {
#pragma unroll
            for (int k = 0; k < V / W; ++k) {
                float x[W];
                unpack_vec<T>(*reinterpret_cast<const typename Raw16<T>::type*>(p + at + k * W), x);
#pragma unroll
                for (int e = 0; e < W; ++e) o[k * W + e] = x[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = to_f32(p[at + e]);
        }
        if (__builtin_amdgcn_ballot_w64(drop > 0 && drop < V)) {
#pragma unroll
            for (int bit = 1; bit < V; bit *= 2)
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = (drop & bit) && e + bit < V ? o[e + bit] : o[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = c + e < C ? to_f32(p[c + e]) : 0.f;
    }
}
template <int V> __device__ __forceinline__ void load_param(const void* p, int dtype, int c, int C, float fill, float (&o)[V]) {
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fill;
    } else if (dtype == 0) load_param_t<float, V>((const float*)p, c, C, o);
    else if (dtype == 1) load_param_t<bf16s, V>((const bf16s*)p, c, C, o);
    else load_param_t<f16s, V>((const f16s*)p, c, C, o);
}
__device__ __forceinline__ void store_param(void* p, int dtype, long at, float v) {
    if (dtype == 0) ((float*)p)[at] = v;
    else if (dtype == 1) ((bf16s*)p)[at] = from_f32<bf16s>(v);
    else ((f16s*)p)[at] = from_f32<f16s>(v);
}

template <int CTRL> __device__ __forceinline__ float dpp_f(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float row16_sum_f(float x) {
    x += dpp_f<0xB1>(x);      // quad_perm [1,0,3,2]
    x += dpp_f<0x4E>(x);      // quad_perm [2,3,0,1]
    x += dpp_f<0x141>(x);     // row_half_mirror
    x += dpp_f<0x140>(x);     // row_mirror
    return x;
}
// x (row16_sum_f's result, or any value per lane) summed over the wave's four rows of 16 lanes, lane by lane
__device__ __forceinline__ float wave_sum_of_rows(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    x = __builtin_bit_cast(float, (unsigned)a[0]) + __builtin_bit_cast(float, (unsigned)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, (unsigned)b[0]) + __builtin_bit_cast(float, (unsigned)b[1]);
}

}  // namespace ppv
