// Multi-head attention, backward (gfx950).  P is computed again from Q, K and the saved log-sum-exp; nothing of size Tq x Tk is stored:
//
//     P = exp2(scale log2e Q K^T - lse),   dP = dO V^T,   D = scale rowsum(dO O),   dS = P (scale dP - D)
//     dQ = dS K,   dK = dS^T Q,   dV = P^T dO
//
// (A row with lse = -inf has no key, or scores of -inf alone: read as +inf it makes P zero in either case, as the forward pass has it.)
// (The scale is in dS when it is rounded to the operands' type: its range in f16 is then that of the results.)
//
// dV's P is rounded to that type as well (in one term or two: attention_tiles.h two_terms).  In f16 weights under 2^-25 would be zero there, and no
// scaled loss could help them: dK / dV computes 2^12 P (one key of e^17.5 times the others' weight over 1500 rows: the others' dV 3.75e-5, else 0),
// takes the 2^12 out of dP and D, which makes dS what it is, and out of dV's sums at the end.
//
// Two launches, no atomics: the gradients have the same bits every time.
//   attn_dq   a wave owns 32 rows (columns of S^T, dP^T, dQ^T) and walks over the keys; it also leaves D for the second launch
//   attn_dkv  a wave owns 32 keys (columns of S, dP, dK^T, dV^T) and walks over the rows of all query heads that share them
// That is 7 products where one launch with atomics on dQ would need 5.  Where few rows (keys) leave the chip idle, the axis that is walked over is
// split; the splits' f32 sums are added in their order by a small launch.  Bound by the matrix pipe and, behind it, the LDS: every operand of a
// tile is read along its rows (S, dP) and across them (dQ, dK, dV).
// Measured (MI355X): 2 x 16 heads of 4096 tokens, D = 128, bf16, causal: dQ 214 us = 960 TFLOP/s, dK / dV 295 us = 930; f32, 32 x 52 rows against
// 1296 keys, 8 heads of 64: 82 and 141 us, the f32 matrix pipe at work in 69 and 59 % of the CUs' busy cycles.
#include "attention_tiles.h"

namespace ppv {

struct AttnBwd {
    AttnDims d;
    AttnTensor q, k, v, g;                                     // g: dO
    const void *out, *out_lo;
    const float* lse;                                          // [B][H][Tq], log2
    float* delta;                                              // [B][H][Tq]: scale rowsum(dO O)
    void *dq, *dk, *dv;
    float* part;                                               // nsplit > 1: f32 sums [nsplit][nbh][rows or Tk][DP] (dK, then dV)
    int ntile, nsplit;
};

__device__ __forceinline__ float lse_or_none(float lse) { return lse == -__builtin_inff() ? __builtin_inff() : lse; }

// a split's share [t0, t1) of the tiles that a workgroup walks over
__device__ __forceinline__ void attn_share(int nsplit, int& t0, int& t1) {
    if (nsplit == 1) return;
    const int per = (t1 - t0 + nsplit - 1) / nsplit;
    t0 = min(t1, t0 + per * (int)blockIdx.y);
    t1 = min(t1, t0 + per);
}

// four waves: OG groups that own 32 columns each x SG groups that divide a staged tile's rows, whose sums meet in LDS at the end
template <class T, int DP, int OG, int ACC> struct BwdShape {
    static constexpr int SG = 4 / OG, KT = 32 * SG;
    static constexpr int NB = 4 * Tile<T, DP>::bytes(KT) <= 81920 ? 2 : 1;
    static constexpr int PARK = (SG - 1) * OG * (DP / 2) * 256 * ACC;
    static constexpr int LDS = 2 * NB * Tile<T, DP>::bytes(KT) > PARK ? 2 * NB * Tile<T, DP>::bytes(KT) : PARK;
    static constexpr int WAVES = DP > 64 && (sizeof(T) == 4 || OG < ACC * 2) ? 1 : DP == 64 && sizeof(T) == 4 && OG <= ACC ? 1 : 2;
};
// adds the other groups' accumulators to the first one's (in their order); false: this wave is done
template <int DB, int OG, int SG> __device__ __forceinline__ bool meet(f32x16* acc, float* lds, int og, int sg, int lane) {
    if constexpr (SG > 1) {
        float* park = lds + og * (SG - 1) * DB * 16 * 64 + lane;
        if (sg > 0)
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) park[((sg - 1) * DB * 16 + i * 16 + j) * 64] = acc[i][j];
        __syncthreads();
        if (sg > 0) return false;
#pragma unroll
        for (int g = 0; g < SG - 1; ++g)
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i][j] += park[(g * DB * 16 + i * 16 + j) * 64];
    }
    return true;
}

template <class T, int DP, int OG>
__global__ __launch_bounds__(256, (BwdShape<T, DP, OG, 1>::WAVES)) void attn_dq_kernel(const AttnBwd a) {
    using TL = Tile<T, DP>;
    using SH = BwdShape<T, DP, OG, 1>;
    constexpr int NT = 256, KT = SH::KT, NB = SH::NB, SG = SH::SG;
    // (keys of few dimensions that a row weighs point the same way, along the row; their part of sum dS K cancels, the roundings of dS do not: with one term dQ
    // was off by 1.52 times a 32-bit computation's error at D = 8.  2 x 16 heads of 4096, D = 32, causal, both directions: 290 -> 310 us)
    constexpr bool TWO = two_terms<T, OG> || (sizeof(T) == 2 && DP == 32);
    __shared__ __attribute__((aligned(16))) char smem[SH::LDS];
    const AttnDims& d = a.d;
    int bh, tile;
    if (!attn_block(d, a.ntile, bh, tile)) return;
    if (d.causal) tile = a.ntile - 1 - tile;
    const int b = bh / d.Hkv, hk = bh - b * d.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, og = wave % OG, sg = wave / OG;
    const int qlen = attn_len(d.q_lens, b, d.Tq), klen = attn_len(d.k_lens, b, d.Tk);
    const int rows = qlen * d.G, shift = klen - qlen;
    const int row0 = tile * OG * 32, row = row0 + og * 32 + (lane & 31);
    const int nch = d.D * TL::ES / 16;
    const RowsOf<T> Q{(const T*)a.q.p + b * a.q.sb + (long)hk * d.G * a.q.sh, a.q.st, a.q.sh, d.G};
    const RowsOf<T> GO{(const T*)a.g.p + b * a.g.sb + (long)hk * d.G * a.g.sh, a.g.st, a.g.sh, d.G};
    const RowsOf<T> K{(const T*)a.k.p + b * a.k.sb + hk * a.k.sh, a.k.st, 0, 1};
    const RowsOf<T> V{(const T*)a.v.p + b * a.v.sb + hk * a.v.sh, a.v.st, 0, 1};

    const int tok = (int)((unsigned)row / (unsigned)d.G), tok0 = (int)((unsigned)row0 / (unsigned)d.G);
    const int last = min(row0 + OG * 32, rows) - 1;
    int kend = klen;
    if (d.causal) kend = min(klen, max(0, (int)((unsigned)max(last, 0) / (unsigned)d.G) + shift + 1));
    if (row0 >= rows) kend = 0;
    int kt0 = 0, kt1 = (kend + KT - 1) / KT;
    attn_share(a.nsplit, kt0, kt1);
    const int lim = row < rows ? (d.causal ? min(klen - 1, tok + shift) : klen - 1) : -1;
    const int lim0 = d.causal ? min(klen - 1, tok0 + shift) : klen - 1;

    using ST = Stager<T, DP, KT, NT>;
    constexpr bool DIRECT = ST::DIRECT && NB == 2;
    const int uwave = __builtin_amdgcn_readfirstlane(wave);
    ST sk, sv;
    auto direct = [&](int kt, int buf) {
        char* t = smem + buf * 2 * TL::bytes(KT);
        ST::direct(t, K, kt * KT, klen, nch, tid, uwave);
        ST::direct(t + TL::bytes(KT), V, kt * KT, klen, nch, tid, uwave);
    };
    if constexpr (DIRECT) {
        if (nch < TL::NCH) {
            clear_lds<4 * TL::bytes(KT), NT>(smem, tid);
            __syncthreads();
        }
        if (kt0 < kt1) direct(kt0, 0);
    } else if (kt0 < kt1) {
        sk.fetch(K, kt0 * KT, klen, nch, tid);
        sv.fetch(V, kt0 * KT, klen, nch, tid);
    }
    u32x4 qf[TL::NF], gf[TL::NF];
    load_own<T, DP>(qf, Q, row, rows, nch, lane);
    load_own<T, DP>(gf, GO, row, rows, nch, lane);
    float delta = 0.f;
    auto dot = [&](const void* out) {
        const RowsOf<T> O{(const T*)out + ((long)b * d.Tq * d.H + hk * d.G) * d.D, (long)d.H * d.D, d.D, d.G};
        u32x4 of[TL::NF];
        load_own<T, DP>(of, O, row, rows, nch, lane);
        float sum = 0.f;
#pragma unroll
        for (int kd = 0; kd < TL::NF; ++kd) {
            float x[16 / TL::ES], y[16 / TL::ES];
            unpack_vec<T>(of[kd], x);
            unpack_vec<T>(gf[kd], y);
#pragma unroll
            for (int e = 0; e < 16 / TL::ES; ++e) sum = __builtin_fmaf(x[e], y[e], sum);
        }
        return sum;
    };
    delta = dot(a.out);
    if (a.out_lo) delta += dot(a.out_lo);                      // O as the forward pass had it: its rounding would be dS's largest error
    delta = half_swap_sum(delta) * d.scale;
    const int h = hk * d.G + (row - tok * d.G);
    const long stat = ((long)b * d.H + h) * d.Tq + tok;
    float lse = 0.f;
    if (row < rows) {
        lse = lse_or_none(a.lse[stat]);
        if (half == 0 && sg == 0 && blockIdx.y == 0) a.delta[stat] = delta;
    }
    const float c = d.scale * LOG2E;
    f32x16 acc[TL::DB];
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;

    const auto L = TL::lane_part(lane);
    const int own = sg * 32;                                   // this group's rows of a tile
    for (int kt = kt0, buf = 0; kt < kt1; ++kt, buf ^= NB - 1) {
        char *tk = smem + buf * 2 * TL::bytes(KT), *tv = tk + TL::bytes(KT);
        if constexpr (DIRECT) {
            wait_direct();
            __syncthreads();
            if (kt + 1 < kt1) direct(kt + 1, buf ^ 1);
        } else {
            if (NB == 1 && kt > kt0) __syncthreads();
            sk.put(tk, tid);
            sv.put(tv, tid);
            __syncthreads();
            if (kt + 1 < kt1) {
                sk.fetch(K, (kt + 1) * KT, klen, nch, tid);
                sv.fetch(V, (kt + 1) * KT, klen, nch, tid);
            }
        }
        __builtin_amdgcn_s_setprio(1);
        f32x16 s, p;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = p[j] = 0.f;
#pragma unroll
        for (int kd = 0; kd < TL::NF; ++kd) {
            s = TL::mma(TL::by_row(tk, L, own, kd), qf[kd], s);
            p = TL::mma(TL::by_row(tv, L, own, kd), gf[kd], p);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], c, -lse)) * __builtin_fmaf(p[j], d.scale, -delta);
        if (__builtin_expect(kt * KT + KT - 1 > lim0, 0)) {    // a key of this tile is hidden from some row
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (kt * KT + own + 8 * (j >> 2) + 4 * half + (j & 3) > lim) s[j] = 0.f;
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kf = 0; kf < TL::CF; ++kf) {
            const u32x4 df = TL::from_acc(s, kf);
            u32x4 dr;
            if constexpr (TWO) dr = TL::rest_of_acc(s, kf, df);
#pragma unroll
            for (int i = 0; i < TL::DB; ++i) {
                const u32x4 kt_ = TL::by_col(tk, L, own, i, kf);
                acc[i] = TL::mma(kt_, df, acc[i]);
                if constexpr (TWO) acc[i] = TL::mma(kt_, dr, acc[i]);
            }
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (SG > 1) __syncthreads();
    if (!meet<TL::DB, OG, SG>(acc, (float*)smem, og, sg, lane)) return;
    if (row >= d.Tq * d.G) return;
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = lim < 0 ? 0.f : acc[i][j];      // (rows that see nothing: zeros, whatever K holds)
    if (a.nsplit > 1) {
        float* po = a.part + (((long)blockIdx.y * d.nbh + bh) * d.Tq * d.G + row) * DP;
#pragma unroll
        for (int i = 0; i < TL::DB; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                store4<float>(po + i * 32 + g * 8 + half * 4, acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]);
        return;
    }
    T* po = (T*)a.dq + (((long)b * d.Tq + tok) * d.H + h) * d.D;
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = i * 32 + g * 8 + half * 4;
            if (e < d.D) store4<T>(po + e, acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]);
        }
}

template <class T, int DP, int OG>
__global__ __launch_bounds__(256, (BwdShape<T, DP, OG, 2>::WAVES)) void attn_dkv_kernel(const AttnBwd a) {
    using TL = Tile<T, DP>;
    using SH = BwdShape<T, DP, OG, 1>;                         // (dK and dV meet one after the other)
    constexpr int NT = 256, QT = SH::KT, NB = SH::NB, SG = SH::SG;
    // K, V, dK, dV of 128 in registers leave one wave per SIMD (328 registers: 430 us where this form took 363, 2 x 16 heads of 4096
    // tokens, causal): V waits in LDS instead
    constexpr bool VL = DP > 64 && sizeof(T) == 2;
    __shared__ __attribute__((aligned(16))) char smem[SH::LDS];
    __shared__ __attribute__((aligned(16))) char vown[VL ? TL::bytes(OG * 32) : 16];
    __shared__ __attribute__((aligned(16))) float stat[NB][2][QT];     // lse, delta
    __shared__ __attribute__((aligned(16))) int limit[NB][QT];         // last key that a row sees
    const AttnDims& d = a.d;
    int bh, tile;
    if (!attn_block(d, a.ntile, bh, tile)) return;
    const int b = bh / d.Hkv, hk = bh - b * d.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, og = wave % OG, sg = wave / OG;
    const int qlen = attn_len(d.q_lens, b, d.Tq), klen = attn_len(d.k_lens, b, d.Tk);
    const int rows = qlen * d.G, shift = klen - qlen;
    const int key0 = tile * OG * 32, key = key0 + og * 32 + (lane & 31);
    const int nch = d.D * TL::ES / 16;
    const RowsOf<T> Q{(const T*)a.q.p + b * a.q.sb + (long)hk * d.G * a.q.sh, a.q.st, a.q.sh, d.G};
    const RowsOf<T> GO{(const T*)a.g.p + b * a.g.sb + (long)hk * d.G * a.g.sh, a.g.st, a.g.sh, d.G};
    const RowsOf<T> K{(const T*)a.k.p + b * a.k.sb + hk * a.k.sh, a.k.st, 0, 1};
    const RowsOf<T> V{(const T*)a.v.p + b * a.v.sb + hk * a.v.sh, a.v.st, 0, 1};

    // rows that see a key of this workgroup
    const int first = d.causal ? max(0, key0 - shift) : 0;     // (token)
    int rt0 = key0 < klen ? (int)min((long)first * d.G, (long)rows) / QT : 0;
    int rt1 = key0 < klen ? (rows + QT - 1) / QT : 0;
    attn_share(a.nsplit, rt0, rt1);

    using ST = Stager<T, DP, QT, NT>;
    constexpr bool DIRECT = ST::DIRECT && NB == 2;
    const int uwave = __builtin_amdgcn_readfirstlane(wave);
    ST sq, so;
    float st = 0.f;
    int sl = -1;
    constexpr float LIFT = __is_same(T, f16s) ? 12.f : 0.f, DOWN = __is_same(T, f16s) ? 0x1p-12f : 1.f;
    if (DIRECT && nch < TL::NCH) {
        clear_lds<DIRECT ? 4 * TL::bytes(QT) : NT * 16, NT>(smem, tid);
        __syncthreads();
    }
    auto fetch = [&](int rt, int buf) {
        if constexpr (DIRECT) {
            char* t = smem + buf * 2 * TL::bytes(QT);
            ST::direct(t, Q, rt * QT, rows, nch, tid, uwave);
            ST::direct(t + TL::bytes(QT), GO, rt * QT, rows, nch, tid, uwave);
        } else {
            sq.fetch(Q, rt * QT, rows, nch, tid);
            so.fetch(GO, rt * QT, rows, nch, tid);
        }
        // the first QT threads: lse and limit; the next QT: delta
        static_assert(2 * QT <= NT && 2 * QT % 64 == 0, "a thread per statistic, whole waves");
        if (uwave < 2 * QT / 64) {
            const int r = rt * QT + tid % QT, rr = min(r, rows - 1), t = d.G == 1 ? rr : (int)((unsigned)rr / (unsigned)d.G);
            st = (tid < QT ? a.lse : a.delta)[((long)b * d.H + hk * d.G + (rr - t * d.G)) * d.Tq + t];
            if (tid < QT) st = lse_or_none(st);
            if constexpr (LIFT != 0.f) st = tid < QT ? st - LIFT : st * DOWN;
            sl = r >= rows ? -1 : d.causal ? min(klen - 1, t + shift) : klen - 1;
        }
    };
    if (rt0 < rt1) fetch(rt0, 0);
    u32x4 kf_[TL::NF], vf[VL ? 1 : TL::NF];
    load_own<T, DP>(kf_, K, key, klen, nch, lane);
    if constexpr (VL) {
        Stager<T, DP, OG * 32, NT> sv;
        sv.fetch(V, key0, klen, nch, tid);
        sv.put(vown, tid);                                     // (the first tile's barrier comes before its first reader)
    } else load_own<T, DP>(vf, V, key, klen, nch, lane);
    const float c = d.scale * LOG2E, scale = d.scale * DOWN;
    f32x16 dk[TL::DB], dv[TL::DB];
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) dk[i][j] = dv[i][j] = 0.f;

    const auto L0 = TL::lane_part(lane);
    const int own = sg * 32;
    for (int rt = rt0, buf = 0; rt < rt1; ++rt, buf ^= NB - 1) {
        char *tq = smem + buf * 2 * TL::bytes(QT), *tg = tq + TL::bytes(QT);
        if (NB == 1 && rt > rt0) __syncthreads();
        if constexpr (DIRECT) wait_direct();
        else {
            sq.put(tq, tid);
            so.put(tg, tid);
        }
        if (tid < 2 * QT) {
            stat[buf][tid / QT][tid % QT] = st;
            if (tid < QT) limit[buf][tid] = sl;
        }
        __syncthreads();
        if (rt + 1 < rt1) fetch(rt + 1, buf ^ 1);
        // (opaque in each turn: the 16 addresses made from it are then computed where they are used and not kept in 16 registers)
        auto L = L0;
        asm volatile("" : "+v"(L.row), "+v"(L.col0), "+v"(L.col1));
        __builtin_amdgcn_s_setprio(1);
        f32x16 s, p;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = p[j] = 0.f;
#pragma unroll
        for (int kd = 0; kd < TL::NF; ++kd) {
            s = TL::mma(TL::by_row(tq, L, own, kd), kf_[kd], s);
            if constexpr (VL) p = TL::mma(TL::by_row(tg, L, own, kd), TL::by_row(vown, L, og * 32, kd), p);
            else p = TL::mma(TL::by_row(tg, L, own, kd), vf[kd], p);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int r = own + 8 * g + 4 * half;
            const float4 ls = *reinterpret_cast<const float4*>(&stat[buf][0][r]), de = *reinterpret_cast<const float4*>(&stat[buf][1][r]);
            const float lsv[4] = {ls.x, ls.y, ls.z, ls.w}, dev[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 4 * g + i;
                const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], c, -lsv[i]));
                s[j] = pe * __builtin_fmaf(p[j], scale, -dev[i]);
                p[j] = pe;
            }
        }
        // a key of this workgroup is hidden from some row of the tile, or the tile is not full
        const int t0 = d.G == 1 ? rt * QT : (int)((unsigned)(rt * QT) / (unsigned)d.G), lim0 = d.causal ? min(klen - 1, t0 + shift) : klen - 1;
        if (__builtin_expect(key0 + OG * 32 - 1 > lim0 || (rt + 1) * QT > rows, 0)) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int4 li = *reinterpret_cast<const int4*>(&limit[buf][own + 8 * g + 4 * half]);
                const int liv[4] = {li.x, li.y, li.z, li.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key > liv[i]) p[4 * g + i] = s[4 * g + i] = 0.f;
            }
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kf = 0; kf < TL::CF; ++kf) {
            const u32x4 pf = TL::from_acc(p, kf), df = TL::from_acc(s, kf);
            u32x4 pr, dr;
            if constexpr (two_terms<T, OG>) {
                pr = TL::rest_of_acc(p, kf, pf);
                dr = TL::rest_of_acc(s, kf, df);
            }
#pragma unroll
            for (int i = 0; i < TL::DB; ++i) {
                const u32x4 gt = TL::by_col(tg, L, own, i, kf), qt = TL::by_col(tq, L, own, i, kf);
                dv[i] = TL::mma(gt, pf, dv[i]);
                dk[i] = TL::mma(qt, df, dk[i]);
                if constexpr (two_terms<T, OG>) {
                    dv[i] = TL::mma(gt, pr, dv[i]);
                    dk[i] = TL::mma(qt, dr, dk[i]);
                }
            }
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (SG > 1) __syncthreads();
    const bool first_group = meet<TL::DB, OG, SG>(dk, (float*)smem, og, sg, lane);
    if (SG > 1) __syncthreads();
    if (!meet<TL::DB, OG, SG>(dv, (float*)smem, og, sg, lane) || !first_group) return;
    if (key >= d.Tk) return;
    if constexpr (LIFT != 0.f)
#pragma unroll
        for (int i = 0; i < TL::DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) dv[i][j] *= DOWN;
    if (a.nsplit > 1) {
        float* pk = a.part + (((long)blockIdx.y * d.nbh + bh) * d.Tk + key) * DP;
        float* pv = pk + (long)a.nsplit * d.nbh * d.Tk * DP;
#pragma unroll
        for (int i = 0; i < TL::DB; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int e = i * 32 + g * 8 + half * 4;
                store4<float>(pk + e, dk[i][4 * g], dk[i][4 * g + 1], dk[i][4 * g + 2], dk[i][4 * g + 3]);
                store4<float>(pv + e, dv[i][4 * g], dv[i][4 * g + 1], dv[i][4 * g + 2], dv[i][4 * g + 3]);
            }
        return;
    }
    const long at = (((long)b * d.Tk + key) * d.Hkv + hk) * d.D;
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = i * 32 + g * 8 + half * 4;
            if (e < d.D) {
                store4<T>((T*)a.dk + at + e, dk[i][4 * g], dk[i][4 * g + 1], dk[i][4 * g + 2], dk[i][4 * g + 3]);
                store4<T>((T*)a.dv + at + e, dv[i][4 * g], dv[i][4 * g + 1], dv[i][4 * g + 2], dv[i][4 * g + 3]);
            }
        }
}

// the splits' sums, added in their order: part [nsplit][nbh][n][DP] -> out; n rows of G heads (dQ) or n keys (G = 1, `heads` = Hkv)
template <class T, int DP> __global__ __launch_bounds__(256) void attn_split_sum_kernel(const float* __restrict__ part, T* __restrict__ out, int nsplit, int nbh,
                                                                                       int Hkv, int G, int n, int D) {
    constexpr int PER = DP / 4;
    const long i = (long)blockIdx.x * 256 + threadIdx.x, at = i / PER;
    const int e = (int)(i % PER) * 4;
    if (at >= (long)nbh * n || e >= D) return;
    float4 s = *reinterpret_cast<const float4*>(part + at * DP + e);
    for (int k = 1; k < nsplit; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(part + ((long)k * nbh * n + at) * DP + e);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    const int bh = (int)(at / n), r = (int)(at % n), b = bh / Hkv, tok = r / G, h = (bh - b * Hkv) * G + (r - tok * G);
    store4<T>(out + (((long)b * (n / G) + tok) * Hkv * G + h) * D + e, s.x, s.y, s.z, s.w);
}

// groups that own rows (keys), tiles of them, ways to split the other axis
struct BwdPlan { int nq, nk, tq, tk, sq, sk, dp; size_t part; };
static BwdPlan attn_bwd_plan(int B, int Hkv, int G, int Tq, int Tk, int D, int es) {
    BwdPlan p;
    p.dp = D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128;
    const int least = es == 4 && p.dp > 64 ? 2 : 1;            // (one group that holds a row's or a key's part of 128 f32 spills)
    auto groups = [&](long n) { return n <= 32 && least == 1 ? 1 : n <= 64 ? 2 : 4; };
    const long rows = (long)Tq * G, bh = (long)B * Hkv;
    p.nq = groups(rows);
    p.nk = groups(Tk);
    p.tq = (int)((rows + p.nq * 32 - 1) / (p.nq * 32));
    p.tk = (Tk + p.nk * 32 - 1) / (p.nk * 32);
    // where the tiles alone leave the chip idle, the other axis is split: at most 512 workgroups, at least four of its tiles each
    auto ways = [&](long base, long walk, int own) {
        long s = base >= 256 ? 1 : 512 / base;
        const long most = walk / (32 * (4 / own)) / 4;
        s = s > most ? most : s;
        return (int)(s < 2 ? 1 : s);
    };
    p.sq = ways(bh * p.tq, Tk, p.nq);
    p.sk = p.tk ? ways(bh * p.tk, rows, p.nk) : 1;
    const size_t q = p.sq > 1 ? (size_t)p.sq * bh * rows * p.dp : 0, k = p.sk > 1 ? (size_t)p.sk * bh * Tk * p.dp * 2 : 0;
    p.part = (q > k ? q : k) * sizeof(float);                  // (dQ's sums are used up before dK's are made)
    return p;
}

template <class T, int DP> static int attn_bwd_t(AttnBwd a, const BwdPlan& p, hipStream_t stream) {
    constexpr int LEAST = sizeof(T) == 4 && DP > 64 ? 2 : 1;
    const AttnDims& d = a.d;
    if (attn_grid(d, p.tq) > ATTN_MAX_GRID || attn_grid(d, p.tk) > ATTN_MAX_GRID) return PPV_ERR_BAD_SIZE;
    auto sum = [&](const float* part, void* out, int nsplit, int G, int n) {
        attn_split_sum_kernel<T, DP><<<(unsigned)(((long)d.nbh * n * (DP / 4) + 255) / 256), 256, 0, stream>>>(part, (T*)out, nsplit, d.nbh, d.Hkv, G, n, d.D);
    };
    a.ntile = p.tq;
    a.nsplit = p.sq;
    dim3 grid((unsigned)attn_grid(d, p.tq), p.sq);
    if (p.nq == 1) attn_dq_kernel<T, DP, LEAST><<<grid, 256, 0, stream>>>(a);
    else if (p.nq == 2) attn_dq_kernel<T, DP, 2><<<grid, 256, 0, stream>>>(a);
    else attn_dq_kernel<T, DP, 4><<<grid, 256, 0, stream>>>(a);
    if (p.sq > 1) sum(a.part, a.dq, p.sq, d.G, d.Tq * d.G);
    if (d.Tk == 0) return ppv_last_error();
    a.ntile = p.tk;
    a.nsplit = p.sk;
    grid = dim3((unsigned)attn_grid(d, p.tk), p.sk);
    if (p.nk == 1) attn_dkv_kernel<T, DP, LEAST><<<grid, 256, 0, stream>>>(a);
    else if (p.nk == 2) attn_dkv_kernel<T, DP, 2><<<grid, 256, 0, stream>>>(a);
    else attn_dkv_kernel<T, DP, 4><<<grid, 256, 0, stream>>>(a);
    if (p.sk > 1) {
        sum(a.part, a.dk, p.sk, 1, d.Tk);
        sum(a.part + (size_t)p.sk * d.nbh * d.Tk * DP, a.dv, p.sk, 1, d.Tk);
    }
    return ppv_last_error();
}
template <class T> static int attn_bwd_dp(const AttnBwd& a, const BwdPlan& p, hipStream_t stream) {
    return p.dp == 32 ? attn_bwd_t<T, 32>(a, p, stream) : p.dp == 64 ? attn_bwd_t<T, 64>(a, p, stream)
         : p.dp == 96 ? attn_bwd_t<T, 96>(a, p, stream) : attn_bwd_t<T, 128>(a, p, stream);
}

}  // namespace ppv

using namespace ppv;

extern "C" {

// delta [B][H][Tq] f32 (rounded up to 16 bytes), then the splits' sums
static size_t delta_bytes(int B, int H, int Tq) { return ((size_t)B * H * Tq * sizeof(float) + 15) / 16 * 16; }

size_t ppv_attention_bwd_workspace_bytes(int B, int H, int Hkv, int Tq, int Tk, int D, int dtype) {
    if (B < 1 || Hkv < 1 || H < Hkv || H % Hkv || Tq < 1 || Tk < 0 || D < 1 || D > 128 || dtype < 0 || dtype > 2) return 0;
    return delta_bytes(B, H, Tq) + attn_bwd_plan(B, Hkv, H / Hkv, Tq, Tk, D, dtype == 0 ? 4 : 2).part;
}

int ppv_attention_bwd(const PpvAttention* x, ppv_stream_t stream) {
    if (!x) return PPV_ERR_NULL;
    AttnBwd a = {};
    if (int e = attn_check(x, &a.d)) return e;
    if (!x->lse || !x->dout || !x->dq || !x->dk || !x->dv) return PPV_ERR_NULL;
    if (!x->workspace) return PPV_ERR_WORKSPACE;
    const int v = x->dtype == 0 ? 4 : 8;
    const long st[] = {x->sgb, x->sgt, x->sgh};
    for (long s : st)
        if (s < 0 || s % v) return PPV_ERR_BAD_SIZE;
    if (x->sgt > 1 << 22) return PPV_ERR_BAD_SIZE;
    const void* ps[] = {x->dout, x->dq, x->dk, x->dv, x->workspace};
    for (const void* p : ps)
        if ((size_t)p % 16) return PPV_ERR_BAD_SIZE;
    a.q = {x->q, x->sqb, x->sqt, x->sqh};
    a.k = {x->k, x->skb, x->skt, x->skh};
    a.v = {x->v, x->svb, x->svt, x->svh};
    a.g = {x->dout, x->sgb, x->sgt, x->sgh};
    a.out = x->out;
    a.out_lo = x->out_lo;
    a.lse = x->lse;
    a.delta = (float*)x->workspace;
    a.part = (float*)((char*)x->workspace + delta_bytes(x->B, x->H, x->Tq));
    const BwdPlan p = attn_bwd_plan(x->B, x->Hkv, a.d.G, x->Tq, x->Tk, x->D, x->dtype == 0 ? 4 : 2);
    a.dq = x->dq;
    a.dk = x->dk;
    a.dv = x->dv;
    return x->dtype == 0 ? attn_bwd_dp<float>(a, p, stream) : x->dtype == 1 ? attn_bwd_dp<bf16s>(a, p, stream) : attn_bwd_dp<f16s>(a, p, stream);
}

}  // extern "C"
