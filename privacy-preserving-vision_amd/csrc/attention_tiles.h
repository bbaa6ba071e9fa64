// What the attention kernels (attention.hip, attention_bwd.hip) share: the problem's description, MFMA fragments for f32, bf16 and f16,
// the layout of a staged tile in LDS.
//
// ROWS.  The query heads that share a key / value head are rows of one problem: row r of (sequence, key head) is token r / G of head
// r % G.  A key tile is then read once for all of them, and dK, dV are sums over rows like any other: no atomics, no second pass.
//
// FRAGMENTS.  Every product is a 32 x 32 tile D[m][n] += A[m][k] B[k][n] whose COLUMNS n are what the wave owns (queries forward and in
// dQ, keys in dK / dV): lane l holds column l % 32 and of its rows 8 g + 4 (l / 32) + r in register 4 g + r.  So a softmax statistic is one
// scalar per lane, and the scores' registers ARE the B operand of the next product, whose k index may run over the rows in any order
// as long as both operands agree: nothing moves between lanes.
//   16-bit: v_mfma_f32_32x32x16, a fragment is 8 elements = 16 bytes a lane; of a product over the tile's rows, fragment kb takes rows
//           16 kb + {0..3, 8..11} (+ 4 in the upper half wave): two transposing LDS reads (ds_read_b64_tr_b16).
//   f32:    v_mfma_f32_32x32x2_f32, four of them per 16-byte fragment; fragment g takes rows 8 g + 0..3 (+ 4).
#pragma once
#include <hip/hip_runtime.h>
#include "elem_types.h"
#include "ppv_common.h"
#include "ppv_hip.h"

namespace ppv {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4_ __attribute__((ext_vector_type(4)));
typedef short s16x8_ __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_ __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_ __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f;

template <class T, int DP> struct Tile {
    static constexpr int ES = sizeof(T);
    static constexpr int DL = DP == 96 ? 128 : DP;             // a staged row's width: 96 lies in rows of 128, the products stop at 96 (2 x 8 heads
                                                               // of 2048, D = 96, bf16, causal, both directions: 191 us, with products of 128 214)
    static constexpr int NCH = DL * ES / 16;                   // 16-byte chunks of a row
    static constexpr int KS = ES == 2 ? 16 : 8;                // k extent of a fragment
    static constexpr int NF = DP / KS;                         // fragments along the head dimension
    static constexpr int CF = 32 / KS;                         // fragments along 32 rows
    static constexpr int DB = DP / 32;                         // 32-wide blocks of the head dimension
    static constexpr int ROW = ES == 2 ? DL * 2 : DL * 4 + 16; // bytes of a staged row
    static constexpr int bytes(int rows) { return rows * ROW; }

    // Where chunk ch of a row lies.  16-bit: XOR with a key of the row's four low bits, chosen so that both readers are free of bank
    // conflicts -- 8 (16) consecutive rows at one chunk (fragments along the head dimension) and 4 rows x 32 (64) bytes (transposing reads)
    // each cover all banks.  f32: an odd number of chunks per row does it.
    static __device__ __forceinline__ int key(int row) {
        const int r0 = row & 1, r1 = (row >> 1) & 1, r2 = (row >> 2) & 1, r3 = (row >> 3) & 1;
        if constexpr (DL == 128) return r2 | r1 << 1 | r0 << 2 | (r1 ^ r3) << 3;
        else if constexpr (DL == 64) return r2 | (r0 ^ r3) << 1 | r1 << 2;
        else return r2 | (r1 ^ r3) << 1;
    }
    static __device__ __forceinline__ int at(int row, int ch) {
        if constexpr (ES == 2) return row * ROW + ((ch ^ key(row)) << 4);
        else return row * ROW + (ch << 4);
    }
    // A lane's own part of the addresses below; what a fragment adds are constants (16-bit: XORed into the chunk bits, which no row stride reaches)
    struct Lane { unsigned row, col0, col1; };
    static __device__ __forceinline__ Lane lane_part(int lane) {
        const int half = lane >> 5, r = 4 * half + ((lane >> 2) & 3), ch = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
        if constexpr (ES == 2)
            return {(unsigned)at(lane & 31, half), (unsigned)(at(r, ch) + (lane & 1) * 8), (unsigned)(at(r + 8, ch) + (lane & 1) * 8)};
        else return {(unsigned)at(lane & 31, half), (unsigned)(4 * half * ROW + (lane & 31) * 4), 0u};
    }
    // A operand with m = row0 + lane % 32, k along the head dimension (fragment kd); row0 a multiple of 16
    static __device__ __forceinline__ u32x4 by_row(const char* tile, const Lane& l, int row0, int kd) {
        const unsigned off = ES == 2 ? l.row ^ (unsigned)(kd << 5) : l.row + (unsigned)(kd << 5);
        return *reinterpret_cast<const u32x4*>(tile + row0 * ROW + off);
    }
    // A operand with m = 32 db + lane % 32 along the head dimension, k over the rows (fragment kf of the 32 rows from row0)
    static __device__ __forceinline__ u32x4 by_col(const char* tile, const Lane& l, int row0, int db, int kf) {
        if constexpr (ES == 2) {
            typedef __attribute__((address_space(3))) s16x4_ lds_s16x4;
            const char* t = tile + (row0 + kf * 16) * ROW;
            const s16x4_ lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t + (l.col0 ^ (unsigned)(db << 6))));
            const s16x4_ hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t + (l.col1 ^ (unsigned)(db << 6))));
            const s16x8_ v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            return __builtin_bit_cast(u32x4, v);
        } else {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const unsigned*>(tile + (row0 + kf * 8 + j) * ROW + db * 128 + l.col0);
            return v;
        }
    }
    // B operand from a product's 16 registers: k over its rows, fragment kf
    static __device__ __forceinline__ u32x4 from_acc(const f32x16& c, int kf) {
        if constexpr (ES == 2) {
            const float v[8] = {c[8 * kf], c[8 * kf + 1], c[8 * kf + 2], c[8 * kf + 3], c[8 * kf + 4], c[8 * kf + 5], c[8 * kf + 6], c[8 * kf + 7]};
            return pack_vec<T>(v);
        } else {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __builtin_bit_cast(unsigned, (float)c[4 * kf + j]);
            return v;
        }
    }
    // what rounding took from from_acc's result, as another fragment of the type
    static __device__ __forceinline__ u32x4 rest_of_acc(const f32x16& c, int kf, u32x4 hi) {
        static_assert(ES == 2, "f32 fragments are the registers themselves");
        float v[8];
        unpack_vec<T>(hi, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c[8 * kf + e] - v[e];
        return pack_vec<T>(v);
    }
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        if constexpr (__is_same(T, bf16s))
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_, a), __builtin_bit_cast(bf16x8_, b), c, 0, 0, 0);
        else if constexpr (__is_same(T, f16s))
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_, a), __builtin_bit_cast(f16x8_, b), c, 0, 0, 0);
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                c = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, (unsigned)a[j]), __builtin_bit_cast(float, (unsigned)b[j]), c, 0, 0, 0);
            return c;
        }
    }
};

// P and dS enter the next product in the operands' 16-bit type.  One term of it is off by half a step (bf16 2^-8, f16 2^-11), which adds to the half step of
// the results' own rounding: 1.35 to 1.45 times the error of a computation in 32 bits that is rounded once.  Two terms (the rounded value and
// what that took) leave the results' rounding alone and cost one more product each.  They are taken where products are not what takes the time: one wave
// owns all rows (keys) of its problem, up to 32, and the walk is bound by the bytes of K and V (Q and dO).  One token of 32 heads on 8, 4 x 65536 keys of
// 128, bf16: 205 us either way; 128 x 32 rows on 1296 keys, 8 heads of 64, both directions: 379 either way.  Where many rows keep the matrix
// pipe busy they would cost a quarter (2 x 16 heads of 4096, D = 32, causal: forward 79 -> 99 us, both directions 297 -> 379).  The dearest
// of what takes them, one token of 88 x 2 heads of 32 on 22456 f16 keys, went from 202 to 213 us.
template <class T, int OG> constexpr bool two_terms = sizeof(T) == 2 && OG == 1;

// The problem, as the kernels take it (elements, not bytes).  Token strides, head strides and batch strides are multiples of 16 bytes.
struct AttnDims {
    int B, H, Hkv, G, Tq, Tk, D, causal;
    const int *q_lens, *k_lens;                                // [B] or null (Tq, Tk)
    float scale;
    int nbh, xcd;                                              // B * Hkv; 1: a (sequence, key head)'s tiles share an XCD
};
struct AttnTensor { const void* p; long sb, st, sh; };
int attn_check(const PpvAttention* x, AttnDims* d);            // (attention.hip)

__device__ __forceinline__ int attn_len(const int* lens, int b, int most) {
    if (!lens) return most;
    const int n = lens[b];
    return n < 0 ? 0 : n > most ? most : n;
}
// blockIdx.x -> (sequence * Hkv + key head, tile).  Workgroups go round the 8 XCDs; with xcd set the tiles of one (sequence, key head) come
// 8 apart, so that one L2 serves them.  Causal tiles differ in length: the first tiles of all heads come first (the caller's tile 0 is the
// longest), then all second ones; head by head the last head's longest tile would start when the others are nearly done.  false: past the end.
__device__ __forceinline__ bool attn_block(const AttnDims& d, int ntile, int& bh, int& tile) {
    const int lanes = d.xcd ? 8 : 1, id = d.xcd ? blockIdx.x >> 3 : blockIdx.x, heads = (d.nbh + lanes - 1) / lanes;
    const int h = d.causal ? id % heads : id / ntile;
    tile = d.causal ? id / heads : id % ntile;
    bh = h * lanes + (d.xcd ? blockIdx.x & 7 : 0);
    return bh < d.nbh;
}
static inline long attn_grid(const AttnDims& d, int ntile) { return (d.xcd ? (d.nbh + 7) / 8 * 8 : d.nbh) * (long)ntile; }
constexpr long ATTN_MAX_GRID = (1 << 24) - 1;                  // workgroups of 256: a launch counts its work items in 32 bits

__device__ __forceinline__ float half_swap_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float half_swap_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// ROWS consecutive rows, NT threads: global -> registers -> LDS.  `row(r)` is row r's address (G = 1 for keys: tokens of one head).  Rows at or
// behind `rows` and chunks behind the head dimension are zeros and are not read.
template <class T> struct RowsOf {
    const T* base;
    long st, sh;
    int G;
    __device__ __forceinline__ const T* row(int r) const {
        if (G == 1) return base + (long)r * st;
        const int t = (int)((unsigned)r / (unsigned)G);
        return base + (long)t * st + (long)(r - t * G) * sh;
    }
};
template <class T, int DP, int ROWS, int NT> struct Stager {
    using TL = Tile<T, DP>;
    static constexpr int ALL = ROWS * TL::NCH, N = (ALL + NT - 1) / NT;
    static constexpr bool EVEN = N * NT == ALL;                // else: more threads than chunks
    static_assert(NT % TL::NCH == 0, "a thread keeps its chunk");
    static constexpr int STEP = NT / TL::NCH;                  // rows from one chunk of a thread to its next
    u32x4 v[N];
    __device__ __forceinline__ void fetch(const RowsOf<T>& src, int row0, int rows, int nch, int tid) {
        const int r0 = tid / TL::NCH, ch = tid % TL::NCH;
        if (src.G == 1 && EVEN && row0 + ROWS <= rows && nch == TL::NCH) {
            // a whole tile: a wave-uniform address and ONE 32-bit offset per lane (the strides are bounded), no lane left out (loads under
            // a condition were waited for one by one: 2.4 of 3.5 us of a dK / dV tile)
            const unsigned off = (unsigned)r0 * (unsigned)src.st * (unsigned)sizeof(T) + (unsigned)ch * 16u;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = *reinterpret_cast<const u32x4*>((const char*)(src.base + (long)(row0 + i * STEP) * src.st) + off);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row0 + i * STEP + r0;
                v[i] = (u32x4){0, 0, 0, 0};
                if (ch < nch && r < rows && (EVEN || i * STEP + r0 < ROWS)) v[i] = *reinterpret_cast<const u32x4*>(src.row(r) + ch * (16 / (int)sizeof(T)));
            }
        }
    }
    __device__ __forceinline__ void put(char* tile, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = i * NT + tid;
            if (EVEN || idx < ALL) *reinterpret_cast<u32x4*>(tile + TL::at(idx / TL::NCH, idx % TL::NCH)) = v[i];
        }
    }

    // The same without registers (16-bit types): whole tiles go from memory to LDS directly, complete after wait_direct() and a barrier.  A
    // wave's 64 lanes fill 1024 consecutive bytes, so it is the SOURCE chunk that is permuted.  Chunks behind the head dimension are not
    // written: the caller has cleared both tile buffers once.  A tile that is not whole goes through registers, zeros behind the end.
    static constexpr bool DIRECT = sizeof(T) == 2 && EVEN && STEP % 16 == 0;
    static __device__ __forceinline__ void direct(char* tile, const RowsOf<T>& src, int row0, int rows, int nch, int tid, int wave) {
        const int r0 = tid / TL::NCH, ch = (tid % TL::NCH) ^ TL::key(r0);                  // (STEP is a multiple of 16: one key for all)
        if (row0 + ROWS <= rows) {
            if (ch < nch) {
                const unsigned off = (unsigned)r0 * (unsigned)src.st * 2u + (unsigned)ch * 16u;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const char* p = src.G == 1 ? (const char*)(src.base + (long)(row0 + i * STEP) * src.st) + off
                                               : (const char*)(src.row(row0 + i * STEP + r0) + ch * 8);
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                                     (__attribute__((address_space(3))) void*)(tile + (i * NT + wave * 64) * 16), 16, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row0 + i * STEP + r0;
                u32x4 x = {0, 0, 0, 0};
                if (ch < nch && r < rows) x = *reinterpret_cast<const u32x4*>(src.row(r) + ch * 8);
                *reinterpret_cast<u32x4*>(tile + (i * NT + tid) * 16) = x;
            }
        }
    }
};
__device__ __forceinline__ void wait_direct() { __builtin_amdgcn_s_waitcnt(0x0F70); }      // vmcnt(0)
template <int BYTES, int NT> __device__ __forceinline__ void clear_lds(char* p, int tid) {
#pragma unroll
    for (int i = 0; i < BYTES / (NT * 16); ++i) *reinterpret_cast<u32x4*>(p + (i * NT + tid) * 16) = (u32x4){0, 0, 0, 0};
    static_assert(BYTES % (NT * 16) == 0, "whole sweeps");
}
// B operand fragments (n = row lane % 32 of 32 rows from row0, k along the head dimension), straight from memory
template <class T, int DP> __device__ __forceinline__ void load_own(u32x4* f, const RowsOf<T>& src, int row, int rows, int nch, int lane) {
    const bool ok = row < rows;
    const T* p = ok ? src.row(row) : src.base;
#pragma unroll
    for (int kd = 0; kd < Tile<T, DP>::NF; ++kd) {
        const int ch = kd * 2 + (lane >> 5);
        f[kd] = ok && ch < nch ? *reinterpret_cast<const u32x4*>(p + ch * (16 / (int)sizeof(T))) : (u32x4){0, 0, 0, 0};
    }
}

// four consecutive results of a lane (registers 4 g .. 4 g + 3) to memory, rounded to T
template <class T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
    else {
        const float v[8] = {a, b, c, d, 0.f, 0.f, 0.f, 0.f};
        const u32x4 r = pack_vec<T>(v);
        *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
    }
}

}  // namespace ppv
