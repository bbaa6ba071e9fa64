// Multi-head attention, forward (gfx950):  S = scale Q K^T,  P = softmax over the visible keys,  O = P V,  and log-sum-exp for the backward pass.
//
// One pass over the keys with a running maximum m and sum l (in units of log2): a tile's P is exp2(S c - m); where m grows, the accumulated O and
// l are scaled by exp2(m_old - m_new).  Neither S nor P reaches memory.  Training and prefill are bound by the matrix pipe and the exponentials,
// a few rows against a long history by the bytes of K and V.
//   * a wave owns 32 rows as the columns of S^T = K Q^T and O^T = V^T P^T (attention_tiles.h): m, l and the scaling are one scalar per
//     lane, P goes from accumulator to operand in place;
//   * a workgroup is four waves, OG row groups x SG key groups (4 x 1, 2 x 2, 1 x 4 for more than 64, more than 32 and up to 32 rows); the
//     key tile staged in LDS is shared by the row groups and divided among the key groups, whose (O, m, l) meet in LDS at the end;
//   * the next tile is on its way during the products: straight into the other LDS buffer (16-bit types), else into registers;
//   * rows behind a sequence's end and rows that see no key are zeros, with -inf; keys behind the end are not read;
//   * few rows and up to 170 tiles of them: the keys are split over workgroups in units of equal length whatever the sequences' lengths, each leaves
//     (O, m, l) in f32, a second launch joins them.
// Measured (MI355X): 2 x 16 heads of 4096 tokens, D = 128, bf16, causal: 155 us = 885 TFLOP/s (a large library product: 1242); of the cycles in
// which the CUs are busy the matrix pipe works in 45 %, the vector ALU in 45 %, and they hardly overlap (the next tile's scores made while this one's
// softmax runs: 163 us and more); one token of 32 heads on
// 8 key heads of 128 against 4 ragged histories of up to 65536: 772 MB in 140-155 us = 5.5-5.0 TB/s, and 6 us for the join; 32 x 52 rows against 1296
// f32 keys, 8 heads of 64: 62 us, the f32 matrix pipe at work in 60 % of them.
#include "attention_tiles.h"

namespace ppv {

struct AttnFwd {
    AttnDims d;
    AttnTensor q, k, v;
    void *out, *out_lo;                                        // [B][Tq][H][D]; out_lo (or null): what rounding took from out
    float* lse;                                                // [B][H][Tq] in units of log2, or null
    float* part;                                               // units: [units][Hkv][rows][DP] f32, then [units][Hkv][rows][2] (m, l)
    int units, ntile;                                          // units = 0: one workgroup has all keys of its rows
};

// The division of all sequences' keys into `units` shares: each is `per` key tiles of one sequence, per as small as the number of shares
// allows (a sequence's last share may be short).  -> units before sequence b (with find >= 0: b is the sequence of unit `find`, -1 if none)
template <int KT> __device__ __forceinline__ void attn_units(const AttnDims& d, int units, int find, int& b, int& first, int& per, int& count) {
    const int lane = threadIdx.x & 63;
    auto tiles = [&](int i) { return i < d.B ? (attn_len(d.k_lens, i, d.Tk) + KT - 1) / KT : 0; };
    int total = 0;
    for (int i = 0; i < d.B; i += 64) {
        int t = tiles(i + lane);
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) t += __shfl_xor(t, s);
        total += t;
    }
    total = __builtin_amdgcn_readfirstlane(total);
    per = max(2, (total + units - d.B - 1) / (units - d.B));   // sum of ceil(t / per) <= total / per + B <= units
    int before = 0;
    for (int i = 0; i < d.B; i += 64) {
        const int n = (tiles(i + lane) + per - 1) / per;
        int upto = n;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o = __shfl_up(upto, s);
            if (lane >= s) upto += o;
        }
        const int from = before + upto - n;
        const unsigned long long hit = __builtin_amdgcn_ballot_w64(find >= 0 ? find >= from && find < from + n : i + lane == b);
        if (hit) {
            const int at = __builtin_ctzll(hit);               // (wave-uniform, and told so: the addresses that follow live in scalar registers)
            b = i + at;
            first = __builtin_amdgcn_readlane(from, at);
            count = __builtin_amdgcn_readlane(n, at);
            return;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (find >= 0) b = -1;
}

template <class T, int DP, int OG> struct FwdShape {
    static constexpr int SG = 4 / OG, MBW = OG == 4 && sizeof(T) == 2 ? 2 : 1, KT = 32 * SG * MBW;
    static constexpr int NB = 4 * Tile<T, DP>::bytes(KT) <= 81920 ? 2 : 1;                 // tile buffers
    static constexpr int PARK = (SG - 1) * OG * (DP / 2 + 2) * 256;                        // where the key groups meet
    static constexpr int LDS = 2 * NB * Tile<T, DP>::bytes(KT) > PARK ? 2 * NB * Tile<T, DP>::bytes(KT) : PARK;
    static constexpr int WAVES = DP > 64 && sizeof(T) == 4 ? 1 : 2;         // per SIMD: 512 or 256 registers
};

// P enters the product with V in the operands' type, in one term or two (attention_tiles.h two_terms).  f16 also has a smallest number:
// beside a largest P of 1 weights under 2^-25 would vanish, and a long history has enough of them to count (65536: 0.2 % of the result; l, in f32, would
// hold them all the same).  There m stays 7 below the running maximum: P up to 2^7, 2^15 with the growth that is let pass, and weights down to 2^-32 count.
template <class T> constexpr float P_LIFT = __is_same(T, f16s) ? 7.f : 0.f;

template <class T, int DP, int OG>
__global__ __launch_bounds__(256, (FwdShape<T, DP, OG>::WAVES)) void attn_fwd_kernel(const AttnFwd a) {
    using TL = Tile<T, DP>;
    using SH = FwdShape<T, DP, OG>;
    constexpr int NT = 256, KT = SH::KT, MBW = SH::MBW, SG = SH::SG, NB = SH::NB;
    __shared__ __attribute__((aligned(16))) char smem[SH::LDS];
    const AttnDims& d = a.d;
    int bh, tile, b, unit = 0, first = 0, per = 0, count = 0;
    if (a.units) {
        tile = blockIdx.x % a.ntile;
        unit = blockIdx.y;
        attn_units<KT>(d, a.units, unit, b, first, per, count);
        if (b < 0) return;
        bh = b * d.Hkv + blockIdx.x / a.ntile;
    } else {
        if (!attn_block(d, a.ntile, bh, tile)) return;
        b = bh / d.Hkv;
    }
    if (d.causal) tile = a.ntile - 1 - tile;                   // the longest first
    const int hk = bh - b * d.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, og = wave % OG, sg = wave / OG;
    const int qlen = attn_len(d.q_lens, b, d.Tq), klen = attn_len(d.k_lens, b, d.Tk);
    const int rows = qlen * d.G, shift = klen - qlen;          // row of token t sees keys up to t + shift where causal
    const int row0 = tile * OG * 32, row = row0 + og * 32 + (lane & 31);
    const int nch = d.D * TL::ES / 16;
    const RowsOf<T> Q{(const T*)a.q.p + b * a.q.sb + (long)hk * d.G * a.q.sh, a.q.st, a.q.sh, d.G};
    const RowsOf<T> K{(const T*)a.k.p + b * a.k.sb + hk * a.k.sh, a.k.st, 0, 1};
    const RowsOf<T> V{(const T*)a.v.p + b * a.v.sb + hk * a.v.sh, a.v.st, 0, 1};

    // keys this workgroup's rows can see, and this unit's share of their tiles
    const int tok = (int)((unsigned)row / (unsigned)d.G), tok0 = (int)((unsigned)row0 / (unsigned)d.G);
    const int last = min(row0 + OG * 32, rows) - 1;
    int kend = klen;
    if (d.causal) kend = min(klen, max(0, (int)((unsigned)max(last, 0) / (unsigned)d.G) + shift + 1));
    if (row0 >= rows) kend = 0;
    int kt0 = 0, kt1 = (kend + KT - 1) / KT;
    if (a.units) {
        kt0 = (unit - first) * per;
        kt1 = min(kt1, kt0 + per);
    }
    const int lim = row < rows ? (d.causal ? min(klen - 1, tok + shift) : klen - 1) : -1;      // last visible key
    const int lim0 = d.causal ? min(klen - 1, tok0 + shift) : klen - 1;                         // ... of the workgroup's first row

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
    u32x4 qf[TL::NF];
    load_own<T, DP>(qf, Q, row, rows, nch, lane);
    f32x16 o[TL::DB];
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    const float c = d.scale * LOG2E;
    const auto L = TL::lane_part(lane);

    for (int kt = kt0, buf = 0; kt < kt1; ++kt, buf ^= NB - 1) {
        char *tk = smem + buf * 2 * TL::bytes(KT), *tv = tk + TL::bytes(KT);
        if constexpr (DIRECT) {
            wait_direct();
            __syncthreads();                                   // this tile is there, and the other buffer's readers are done
            if (kt + 1 < kt1) direct(kt + 1, buf ^ 1);
        } else {
            if (NB == 1 && kt > kt0) __syncthreads();          // (with two buffers the other one's readers passed the barrier of the tile before)
            sk.put(tk, tid);
            sv.put(tv, tid);
            __syncthreads();
            if (kt + 1 < kt1) {
                sk.fetch(K, (kt + 1) * KT, klen, nch, tid);
                sv.fetch(V, (kt + 1) * KT, klen, nch, tid);
            }
        }
        const int own = sg * MBW * 32;                         // this key group's rows of the tile
        __builtin_amdgcn_s_setprio(1);
        f32x16 s[MBW];
#pragma unroll
        for (int mb = 0; mb < MBW; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[mb][j] = 0.f;
#pragma unroll
        for (int kd = 0; kd < TL::NF; ++kd)
#pragma unroll
            for (int mb = 0; mb < MBW; ++mb) s[mb] = TL::mma(TL::by_row(tk, L, own + mb * 32, kd), qf[kd], s[mb]);
        __builtin_amdgcn_s_setprio(0);
        if (__builtin_expect(kt * KT + KT - 1 > lim0, 0)) {    // a key of this tile is hidden from some row
#pragma unroll
            for (int mb = 0; mb < MBW; ++mb)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (kt * KT + own + mb * 32 + 8 * (j >> 2) + 4 * half + (j & 3) > lim) s[mb][j] = -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int mb = 0; mb < MBW; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, s[mb][j]);
        top = half_swap_max(top) * c;
        // The running maximum follows only where it has grown by more than 2^8 (P, l and O then stay below 256 times what they would be: nothing
        // to f32, and P's rounding is relative; 2^15 is in f16's range).  Without the hint the branch becomes 64 products and 64 copies in every tile.
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m + (8.f + P_LIFT<T>)) != 0, 0)) {
            const float mn = fmaxf(m, top - P_LIFT<T>), alpha = __builtin_amdgcn_exp2f(mn == -__builtin_inff() ? 0.f : m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < TL::DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= alpha;
        }
        const float mu = m == -__builtin_inff() ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int mb = 0; mb < MBW; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                s[mb][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mb][j], c, -mu));
                sum += s[mb][j];
            }
        l += sum;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int mb = 0; mb < MBW; ++mb)
#pragma unroll
            for (int kf = 0; kf < TL::CF; ++kf) {
                const u32x4 pf = TL::from_acc(s[mb], kf);
                u32x4 pr;
                if constexpr (two_terms<T, OG>) pr = TL::rest_of_acc(s[mb], kf, pf);
#pragma unroll
                for (int i = 0; i < TL::DB; ++i) {
                    const u32x4 vt = TL::by_col(tv, L, own + mb * 32, i, kf);
                    o[i] = TL::mma(vt, pf, o[i]);
                    if constexpr (two_terms<T, OG>) o[i] = TL::mma(vt, pr, o[i]);
                }
            }
        __builtin_amdgcn_s_setprio(0);
    }
    l = half_swap_sum(l);
    if constexpr (SG > 1) {                                    // the key groups' shares of the same rows, added in their order
        __syncthreads();
        float* park = (float*)smem + og * (SG - 1) * (DP / 2 + 2) * 64 + lane;
        if (sg > 0) {
            float* p = park + (sg - 1) * (DP / 2 + 2) * 64;
            p[0] = m;
            p[64] = l;
#pragma unroll
            for (int i = 0; i < TL::DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) p[(2 + i * 16 + j) * 64] = o[i][j];
        }
        __syncthreads();
        if (sg > 0) return;
        float mn = m;
#pragma unroll
        for (int g = 0; g < SG - 1; ++g) mn = fmaxf(mn, park[g * (DP / 2 + 2) * 64]);
        const float mu = mn == -__builtin_inff() ? 0.f : mn, w0 = __builtin_amdgcn_exp2f(m - mu);
        m = mn;
        l *= w0;
#pragma unroll
        for (int i = 0; i < TL::DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] *= w0;
#pragma unroll
        for (int g = 0; g < SG - 1; ++g) {
            const float* p = park + g * (DP / 2 + 2) * 64;
            const float w = __builtin_amdgcn_exp2f(p[0] - mu);
            l = __builtin_fmaf(w, p[64], l);
#pragma unroll
            for (int i = 0; i < TL::DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] = __builtin_fmaf(w, p[(2 + i * 16 + j) * 64], o[i][j]);
        }
    }
    if (lim < 0) l = 0.f;                                      // (a row that sees nothing may have gone through tiles that its neighbours see)
    if (l == 0.f) {
        m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < TL::DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    }

    const int whole = d.Tq * d.G;                              // rows of the result: those behind the sequence's end are zeros
    if (row >= whole) return;
    if (a.units) {
        const long at = ((long)unit * d.Hkv + hk) * whole + row;
        float* ml = a.part + (long)a.units * d.Hkv * whole * DP + at * 2;
        if (half == 0) { ml[0] = m; ml[1] = l; }
        float* po = a.part + at * DP;
#pragma unroll
        for (int i = 0; i < TL::DB; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                store4<float>(po + i * 32 + g * 8 + half * 4, o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int h = hk * d.G + (row - tok * d.G);
    const long at = (((long)b * d.Tq + tok) * d.H + h) * d.D;
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = i * 32 + g * 8 + half * 4;
            if (e < d.D) {
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = o[i][4 * g + r] * inv;
                store4<T>((T*)a.out + at + e, x[0], x[1], x[2], x[3]);
                if (a.out_lo) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] -= to_f32(from_f32<T>(x[r]));
                    store4<T>((T*)a.out_lo + at + e, x[0], x[1], x[2], x[3]);
                }
            }
        }
    if (a.lse && half == 0)
        a.lse[((long)b * d.H + h) * d.Tq + tok] = l == 0.f ? -__builtin_inff() : m + __builtin_amdgcn_logf(l);
}

// joins a row's units: O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s; a wave per row
template <class T, int DP, int KT> __global__ __launch_bounds__(256) void attn_join_kernel(const AttnFwd a) {
    const AttnDims& d = a.d;
    const int whole = d.Tq * d.G, lane = threadIdx.x & 63;
    const long n = (long)d.Hkv * whole, at = (long)blockIdx.x * 4 + (threadIdx.x >> 6);       // rows of one sequence
    int b = blockIdx.y, first = 0, per = 0, count = 0;
    attn_units<KT>(d, a.units, -1, b, first, per, count);
    if (at >= n) return;
    const float* ml = a.part + (long)a.units * n * DP;
    constexpr int E = (DP + 63) / 64;
    float o[E], l = 0.f, m = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int s = lane; s < count; s += 64) m = fmaxf(m, ml[((first + s) * n + at) * 2]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
    const float mu = m == -__builtin_inff() ? 0.f : m;
    for (int s0 = 0; s0 < count; s0 += 64) {
        const long u = (first + s0 + lane) * n + at;
        const bool some = s0 + lane < count;
        const float w = some ? __builtin_amdgcn_exp2f(ml[u * 2] - mu) : 0.f;
        float lw = some ? w * ml[u * 2 + 1] : 0.f;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) lw += __shfl_xor(lw, s);
        l += lw;
        const int here = min(64, count - s0);
        for (int s = 0; s < here; s += 8) {                    // eight units' loads at a time
            float x[8][E];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float* po = a.part + ((first + s0 + min(s + i, here - 1)) * n + at) * DP;
#pragma unroll
                for (int e = 0; e < E; ++e) x[i][e] = po[min(lane + 64 * e, DP - 1)];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float ws = s + i < here ? __shfl(w, s + i) : 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(ws, x[i][e], o[e]);
            }
        }
    }
    const int hk = (int)(at / whole), row = (int)(at - (long)hk * whole), tok = row / d.G, h = hk * d.G + (row - tok * d.G);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const long to = (((long)b * d.Tq + tok) * d.H + h) * d.D;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < d.D) {
            const float x = o[e] * inv;
            const T r = from_f32<T>(x);
            ((T*)a.out)[to + lane + 64 * e] = r;
            if (a.out_lo) ((T*)a.out_lo)[to + lane + 64 * e] = from_f32<T>(x - to_f32(r));
        }
    if (a.lse && lane == 0) a.lse[((long)b * d.H + h) * d.Tq + tok] = l == 0.f ? -__builtin_inff() : m + __builtin_amdgcn_logf(l);
}

// row groups of a workgroup, its tiles, shares of the keys
struct AttnPlan { int og, ntile, dp; long units; };
static AttnPlan attn_fwd_plan(int B, int Hkv, int G, int Tq, int Tk, int D, int es) {
    AttnPlan p;
    const long rows = (long)Tq * G;
    p.dp = D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128;
    p.og = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
    p.ntile = (int)((rows + p.og * 32 - 1) / (p.og * 32));
    // split where the tiles alone are fewer than a third of what is resident (one token, 8 key heads of 128, bf16, B sequences of 16384 keys: 168 tiles,
    // split, 4.55 TB/s; 176 to 512, each a walk over its whole sequence, 4.7 to 5.8.  With lengths from a quarter to the whole 4.5 split, but 3.2 for 176, 4.3
    // for 256 and 5.0 for 512 tiles, where the longest walk ends alone): at most 512 workgroups (two for each CU, all of them resident: with 544 the last
    // 32 of a history of 65536 keys ran alone, 179 us instead of 149), with at least two key tiles each
    const long base = (long)B * Hkv * p.ntile, kt = p.og == 4 ? (es == 2 ? 64 : 32) : p.og == 2 ? 64 : 128, ktiles = (Tk + kt - 1) / kt;
    long s = base >= 256 ? 1 : 512 / base - 1;
    s = s > ktiles / 2 ? ktiles / 2 : s;
    p.units = s < 2 ? 0 : s * B + B;                           // (B of them for the sequences' short last shares)
    return p;
}

template <class T, int DP, int OG> static void attn_fwd_og(const AttnFwd& a, hipStream_t stream) {
    if (!a.units) {
        attn_fwd_kernel<T, DP, OG><<<(unsigned)attn_grid(a.d, a.ntile), 256, 0, stream>>>(a);
        return;
    }
    attn_fwd_kernel<T, DP, OG><<<dim3(a.d.Hkv * a.ntile, a.units), 256, 0, stream>>>(a);
    attn_join_kernel<T, DP, FwdShape<T, DP, OG>::KT><<<dim3((unsigned)(((long)a.d.Hkv * a.d.Tq * a.d.G + 3) / 4), a.d.B), 256, 0, stream>>>(a);
}
template <class T, int DP> static int attn_fwd_t(const AttnFwd& a, const AttnPlan& p, hipStream_t stream) {
    if (p.og == 1) attn_fwd_og<T, DP, 1>(a, stream);
    else if (p.og == 2) attn_fwd_og<T, DP, 2>(a, stream);
    else attn_fwd_og<T, DP, 4>(a, stream);
    return ppv_last_error();
}
template <class T> static int attn_fwd_dp(const AttnFwd& a, const AttnPlan& p, hipStream_t stream) {
    return p.dp == 32 ? attn_fwd_t<T, 32>(a, p, stream) : p.dp == 64 ? attn_fwd_t<T, 64>(a, p, stream)
         : p.dp == 96 ? attn_fwd_t<T, 96>(a, p, stream) : attn_fwd_t<T, 128>(a, p, stream);
}

// the checks that both directions share; 0 or an error
int attn_check(const PpvAttention* x, AttnDims* d) {
    const int es = x->dtype == 0 ? 4 : 2, v = 16 / es;
    if (!x->q || !x->k || !x->v || !x->out) return PPV_ERR_NULL;
    if (x->dtype < 0 || x->dtype > 2 || x->B < 1 || x->H < 1 || x->Hkv < 1 || x->H % x->Hkv || x->Tq < 1 || x->Tk < 0 || x->D < 1 || x->D > 128 ||
        x->D % v || !(x->scale > 0.f) || x->scale > 1e30f)
        return PPV_ERR_BAD_SIZE;
    if ((long)x->Tq * (x->H / x->Hkv) > 0x3fffffffL || x->Tk > 0x3fffffff || (long)x->B * x->Hkv > 0x3fffffffL) return PPV_ERR_BAD_SIZE;
    if ((long)x->B * ((x->Tk + 31L) / 32) > 0x3fffffffL) return PPV_ERR_BAD_SIZE;              // (key tiles of all sequences are counted in 32 bits)
    const long st[] = {x->sqb, x->sqt, x->sqh, x->skb, x->skt, x->skh, x->svb, x->svt, x->svh};
    for (long s : st)
        if (s < 0 || s % v) return PPV_ERR_BAD_SIZE;
    if (x->sqt > 1 << 22 || x->skt > 1 << 22 || x->svt > 1 << 22) return PPV_ERR_BAD_SIZE;      // (offsets inside a tile are 32 bits)
    const void* ps[] = {x->q, x->k, x->v, x->out, x->out_lo};
    for (const void* p : ps)
        if ((size_t)p % 16) return PPV_ERR_BAD_SIZE;
    *d = {x->B, x->H, x->Hkv, x->H / x->Hkv, x->Tq, x->Tk, x->D, x->causal != 0, x->q_lens, x->k_lens, x->scale, x->B * x->Hkv, 0};
    d->xcd = d->nbh % 8 == 0 || d->nbh >= 64;
    return PPV_OK;
}

}  // namespace ppv

using namespace ppv;

extern "C" {

size_t ppv_attention_fwd_workspace_bytes(int B, int H, int Hkv, int Tq, int Tk, int D, int dtype) {
    if (B < 1 || Hkv < 1 || H < Hkv || H % Hkv || Tq < 1 || Tk < 0 || D < 1 || D > 128 || dtype < 0 || dtype > 2) return 0;
    const AttnPlan p = attn_fwd_plan(B, Hkv, H / Hkv, Tq, Tk, D, dtype == 0 ? 4 : 2);
    return (size_t)p.units * H * Tq * (p.dp + 2) * sizeof(float);
}

int ppv_attention_fwd(const PpvAttention* x, ppv_stream_t stream) {
    if (!x) return PPV_ERR_NULL;
    AttnFwd a = {};
    if (int e = attn_check(x, &a.d)) return e;
    const AttnPlan p = attn_fwd_plan(x->B, x->Hkv, a.d.G, x->Tq, x->Tk, x->D, x->dtype == 0 ? 4 : 2);
    if (p.units && !x->workspace) return PPV_ERR_WORKSPACE;
    if (attn_grid(a.d, p.ntile) > ATTN_MAX_GRID || (p.units && (size_t)x->workspace % 16)) return PPV_ERR_BAD_SIZE;
    a.q = {x->q, x->sqb, x->sqt, x->sqh};
    a.k = {x->k, x->skb, x->skt, x->skh};
    a.v = {x->v, x->svb, x->svt, x->svh};
    a.out = x->out;
    a.lse = x->lse;
    a.part = (float*)x->workspace;
    a.units = (int)p.units;
    a.out_lo = x->out_lo;
    a.ntile = p.ntile;
    return x->dtype == 0 ? attn_fwd_dp<float>(a, p, stream) : x->dtype == 1 ? attn_fwd_dp<bf16s>(a, p, stream) : attn_fwd_dp<f16s>(a, p, stream);
}

}  // extern "C"
