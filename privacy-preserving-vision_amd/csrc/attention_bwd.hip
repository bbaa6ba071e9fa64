// Multi-head attention, backward (gfx950).  P is computed again from Q, K and the saved log-sum-exp; nothing of size Tq x Tk is stored:
//
//     P = exp2(scale log2e Q K^T - lse),   dP = dO V^T,   D = rowsum(dO O),   dS = P (dP - D)
//     dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
//
// Two launches, no atomics: the gradients have the same bits every time.
//   attn_dq   a wave owns 32 rows (columns of S^T, dP^T, dQ^T) and walks over the keys; it also leaves D for the second launch
//   attn_dkv  a wave owns 32 keys (columns of S, dP, dK^T, dV^T) and walks over the rows of all query heads that share them
// That is 7 products where one launch with atomics on dQ would need 5.  Bound by the matrix pipe and, behind it, the LDS: every operand of a
// tile is read along its rows (S, dP) and across them (dQ, dK, dV).
#include "attention_tiles.h"

namespace ppv {

struct AttnBwd {
    AttnDims d;
    AttnTensor q, k, v, g;                                     // g: dO
    const void *out, *out_lo;
    const float* lse;                                          // [B][H][Tq], log2
    float* delta;                                              // [B][H][Tq]
    void *dq, *dk, *dv;
    int ntile;
};

// four waves: OG groups that own 32 columns each x SG groups that divide a staged tile's rows, whose sums meet in LDS at the end
template <class T, int DP, int OG, int ACC> struct BwdShape {
    static constexpr int SG = 4 / OG, KT = 32 * SG;
    static constexpr int NB = 4 * Tile<T, DP>::bytes(KT) <= 65536 ? 2 : 1;
    static constexpr int PARK = (SG - 1) * OG * (DP / 2) * 256 * ACC;
    static constexpr int LDS = 2 * NB * Tile<T, DP>::bytes(KT) > PARK ? 2 * NB * Tile<T, DP>::bytes(KT) : PARK;
    static constexpr int WAVES = DP == 128 && (sizeof(T) == 4 || OG < ACC * 2) ? 1 : DP == 64 && sizeof(T) == 4 && OG <= ACC ? 1 : 2;
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
    const int ktiles = (kend + KT - 1) / KT;
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
        if (ktiles) direct(0, 0);
    } else if (ktiles) {
        sk.fetch(K, 0, klen, nch, tid);
        sv.fetch(V, 0, klen, nch, tid);
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
    delta = half_swap_sum(delta);
    const int h = hk * d.G + (row - tok * d.G);
    const long stat = ((long)b * d.H + h) * d.Tq + tok;
    float lse = 0.f;
    if (row < rows) {
        lse = a.lse[stat];
        if (half == 0 && sg == 0) a.delta[stat] = delta;
    }
    const float c = d.scale * LOG2E;
    f32x16 acc[TL::DB];
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;

    const auto L = TL::lane_part(lane);
    const int own = sg * 32;                                   // this group's rows of a tile
    for (int kt = 0, buf = 0; kt < ktiles; ++kt, buf ^= NB - 1) {
        char *tk = smem + buf * 2 * TL::bytes(KT), *tv = tk + TL::bytes(KT);
        if constexpr (DIRECT) {
            wait_direct();
            __syncthreads();
            if (kt + 1 < ktiles) direct(kt + 1, buf ^ 1);
        } else {
            if (NB == 1 && kt > 0) __syncthreads();
            sk.put(tk, tid);
            sv.put(tv, tid);
            __syncthreads();
            if (kt + 1 < ktiles) {
                sk.fetch(K, (kt + 1) * KT, klen, nch, tid);
                sv.fetch(V, (kt + 1) * KT, klen, nch, tid);
            }
        }
        f32x16 s, p;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = p[j] = 0.f;
#pragma unroll
        for (int kd = 0; kd < TL::NF; ++kd) {
            s = TL::mma(TL::by_row(tk, L, own, kd), qf[kd], s);
            p = TL::mma(TL::by_row(tv, L, own, kd), gf[kd], p);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], c, -lse)) * (p[j] - delta);
        if (__builtin_expect(kt * KT + KT - 1 > lim0, 0)) {    // a key of this tile is hidden from some row
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (kt * KT + own + 8 * (j >> 2) + 4 * half + (j & 3) > lim) s[j] = 0.f;
        }
#pragma unroll
        for (int kf = 0; kf < TL::CF; ++kf) {
            const u32x4 df = TL::from_acc(s, kf);
#pragma unroll
            for (int i = 0; i < TL::DB; ++i) acc[i] = TL::mma(TL::by_col(tk, L, own, i, kf), df, acc[i]);
        }
    }
    if (SG > 1) __syncthreads();
    if (!meet<TL::DB, OG, SG>(acc, (float*)smem, og, sg, lane)) return;
    if (row >= d.Tq * d.G) return;
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = lim < 0 ? 0.f : acc[i][j] * d.scale;      // (rows that see nothing: zeros, whatever K holds)
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
    // K, V, dK, dV of 128 in registers leave one wave per SIMD (328 registers: 580 us where this form takes 390, 2 x 16 heads of 4096
    // tokens, causal): V waits in LDS instead
    constexpr bool VL = DP == 128 && sizeof(T) == 2;
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
    const int rt0 = key0 < klen ? (int)min((long)first * d.G, (long)rows) / QT : 0;
    const int rt1 = key0 < klen ? (rows + QT - 1) / QT : 0;

    using ST = Stager<T, DP, QT, NT>;
    constexpr bool DIRECT = ST::DIRECT && NB == 2;
    const int uwave = __builtin_amdgcn_readfirstlane(wave);
    ST sq, so;
    float st = 0.f;
    int sl = -1;
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
    const float c = d.scale * LOG2E;
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
        f32x16 s, p;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = p[j] = 0.f;
#pragma unroll
        for (int kd = 0; kd < TL::NF; ++kd) {
            s = TL::mma(TL::by_row(tq, L, own, kd), kf_[kd], s);
            if constexpr (VL) p = TL::mma(TL::by_row(tg, L, own, kd), TL::by_row(vown, L, og * 32, kd), p);
            else p = TL::mma(TL::by_row(tg, L, own, kd), vf[kd], p);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int r = own + 8 * g + 4 * half;
            const float4 ls = *reinterpret_cast<const float4*>(&stat[buf][0][r]), de = *reinterpret_cast<const float4*>(&stat[buf][1][r]);
            const float lsv[4] = {ls.x, ls.y, ls.z, ls.w}, dev[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 4 * g + i;
                const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], c, -lsv[i]));
                s[j] = pe * (p[j] - dev[i]);
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
#pragma unroll
        for (int kf = 0; kf < TL::CF; ++kf) {
            const u32x4 pf = TL::from_acc(p, kf), df = TL::from_acc(s, kf);
#pragma unroll
            for (int i = 0; i < TL::DB; ++i) {
                dv[i] = TL::mma(TL::by_col(tg, L, own, i, kf), pf, dv[i]);
                dk[i] = TL::mma(TL::by_col(tq, L, own, i, kf), df, dk[i]);
            }
        }
    }
    if (SG > 1) __syncthreads();
    const bool first_group = meet<TL::DB, OG, SG>(dk, (float*)smem, og, sg, lane);
    if (SG > 1) __syncthreads();
    if (!meet<TL::DB, OG, SG>(dv, (float*)smem, og, sg, lane) || !first_group) return;
    if (key >= d.Tk) return;
    const long at = (((long)b * d.Tk + key) * d.Hkv + hk) * d.D;
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = i * 32 + g * 8 + half * 4;
            if (e < d.D) {
                store4<T>((T*)a.dk + at + e, dk[i][4 * g] * d.scale, dk[i][4 * g + 1] * d.scale, dk[i][4 * g + 2] * d.scale, dk[i][4 * g + 3] * d.scale);
                store4<T>((T*)a.dv + at + e, dv[i][4 * g], dv[i][4 * g + 1], dv[i][4 * g + 2], dv[i][4 * g + 3]);
            }
        }
}

static int attn_groups(long n) { return n <= 32 ? 1 : n <= 64 ? 2 : 4; }

template <class T, int DP> static int attn_bwd_t(AttnBwd a, hipStream_t stream) {
    const long rows = (long)a.d.Tq * a.d.G;
    constexpr int LEAST = sizeof(T) == 4 && DP == 128 ? 2 : 1;  // (one group that holds a row's or a key's part of 128 f32 spills)
    const int nq = attn_groups(rows) < LEAST ? LEAST : attn_groups(rows), nk = attn_groups(a.d.Tk) < LEAST ? LEAST : attn_groups(a.d.Tk);
    a.ntile = (int)((rows + nq * 32 - 1) / (nq * 32));
    const int tk = (a.d.Tk + nk * 32 - 1) / (nk * 32);
    if ((long)a.d.nbh * a.ntile > 0x7ffffff0L || (long)a.d.nbh * tk > 0x7ffffff0L) return PPV_ERR_BAD_SIZE;
    unsigned grid = attn_grid(a.d, a.ntile);
    if (nq == 1) attn_dq_kernel<T, DP, LEAST><<<grid, 256, 0, stream>>>(a);
    else if (nq == 2) attn_dq_kernel<T, DP, 2><<<grid, 256, 0, stream>>>(a);
    else attn_dq_kernel<T, DP, 4><<<grid, 256, 0, stream>>>(a);
    if (a.d.Tk == 0) return ppv_last_error();
    a.ntile = tk;
    grid = attn_grid(a.d, tk);
    if (nk == 1) attn_dkv_kernel<T, DP, LEAST><<<grid, 256, 0, stream>>>(a);
    else if (nk == 2) attn_dkv_kernel<T, DP, 2><<<grid, 256, 0, stream>>>(a);
    else attn_dkv_kernel<T, DP, 4><<<grid, 256, 0, stream>>>(a);
    return ppv_last_error();
}
template <class T> static int attn_bwd_dp(const AttnBwd& a, hipStream_t stream) {
    return a.d.D <= 32 ? attn_bwd_t<T, 32>(a, stream) : a.d.D <= 64 ? attn_bwd_t<T, 64>(a, stream) : attn_bwd_t<T, 128>(a, stream);
}

}  // namespace ppv

using namespace ppv;

extern "C" {

size_t ppv_attention_bwd_workspace_bytes(int B, int H, int Tq) {
    return B < 1 || H < 1 || Tq < 1 ? 0 : (size_t)B * H * Tq * sizeof(float);
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
    const void* ps[] = {x->dout, x->dq, x->dk, x->dv};
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
    a.dq = x->dq;
    a.dk = x->dk;
    a.dv = x->dv;
    return x->dtype == 0 ? attn_bwd_dp<float>(a, stream) : x->dtype == 1 ? attn_bwd_dp<bf16s>(a, stream) : attn_bwd_dp<f16s>(a, stream);
}

}  // extern "C"
