// Multi-head attention, forward (gfx950):  S = scale Q K^T,  P = softmax over the visible keys,  O = P V,  and log-sum-exp for the backward pass.
//
// One pass over the keys with a running maximum m and sum l (in units of log2): a tile's P is exp2(S c - m), the accumulated O and l are
// scaled by exp2(m_old - m_new).  Neither S nor P reaches memory.  Training and prefill are bound by the matrix pipe and the exponentials,
// a few rows against a long history by the bytes of K and V.
//   * a wave owns 32 rows as the columns of S^T = K Q^T and O^T = V^T P^T (attention_tiles.h): m, l and the scaling are one scalar per
//     lane, P goes from accumulator to operand in place;
//   * a workgroup's NW waves share key tiles staged in LDS, double-buffered, the next one in registers during the products;
//   * rows behind a sequence's end and rows that see no key are zeros, with -inf; keys behind the end are not read;
//   * few rows: the keys are split over workgroups, each leaves (O, m, l) in f32, a second launch joins them.
#include "attention_tiles.h"

namespace ppv {

struct AttnFwd {
    AttnDims d;
    AttnTensor q, k, v;
    void* out;                                                 // [B][Tq][H][D]
    float* lse;                                                // [B][H][Tq] in units of log2, or null
    float* part;                                               // split: [nsplit][nbh][rows][DP] f32, then [nsplit][nbh][rows][2] (m, l)
    int nsplit, ntile;
};

template <class T, int DP, int NW, int KT>
__global__ __launch_bounds__(NW * 64) void attn_fwd_kernel(const AttnFwd a) {
    using TL = Tile<T, DP>;
    constexpr int NT = NW * 64, MB = KT / 32;
    __shared__ __attribute__((aligned(16))) char smem[2][2][TL::bytes(KT)];
    const AttnDims& d = a.d;
    int bh, tile;
    if (!attn_block(d, a.ntile, bh, tile)) return;
    if (d.causal) tile = a.ntile - 1 - tile;                   // the longest first
    const int b = bh / d.Hkv, hk = bh - b * d.Hkv, split = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int qlen = attn_len(d.q_lens, b, d.Tq), klen = attn_len(d.k_lens, b, d.Tk);
    const int rows = qlen * d.G, shift = klen - qlen;          // row of token t sees keys up to t + shift where causal
    const int row0 = tile * NW * 32, row = row0 + wave * 32 + (lane & 31);
    const int nch = d.D * TL::ES / 16;
    const RowsOf<T> Q{(const T*)a.q.p + b * a.q.sb + (long)hk * d.G * a.q.sh, a.q.st, a.q.sh, d.G};
    const RowsOf<T> K{(const T*)a.k.p + b * a.k.sb + hk * a.k.sh, a.k.st, 0, 1};
    const RowsOf<T> V{(const T*)a.v.p + b * a.v.sb + hk * a.v.sh, a.v.st, 0, 1};

    // keys this workgroup's rows can see, and this split's share of their tiles
    const int tok = (int)((unsigned)row / (unsigned)d.G), tok0 = (int)((unsigned)row0 / (unsigned)d.G);
    const int last = min(row0 + NW * 32, rows) - 1;
    int kend = klen;
    if (d.causal) kend = min(klen, max(0, (int)((unsigned)max(last, 0) / (unsigned)d.G) + shift + 1));
    if (row0 >= rows) kend = 0;
    const int ktiles = (kend + KT - 1) / KT, per = (ktiles + a.nsplit - 1) / a.nsplit;
    const int kt0 = split * per, kt1 = min(ktiles, kt0 + per);
    const int lim = row < rows ? (d.causal ? min(klen - 1, tok + shift) : klen - 1) : -1;      // last visible key
    const int lim0 = d.causal ? min(klen - 1, tok0 + shift) : klen - 1;                         // ... of the workgroup's first row

    u32x4 qf[TL::NF];
    load_own<T, DP>(qf, Q, row, rows, nch, lane);
    f32x16 o[TL::DB];
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    const float c = d.scale * LOG2E;

    Stager<T, DP, KT, NT> sk, sv;
    if (kt0 < kt1) {
        sk.fetch(K, kt0 * KT, klen, nch, tid);
        sv.fetch(V, kt0 * KT, klen, nch, tid);
    }
    for (int kt = kt0, buf = 0; kt < kt1; ++kt, buf ^= 1) {
        char *tk = smem[buf][0], *tv = smem[buf][1];
        sk.put(tk, tid);
        sv.put(tv, tid);
        __syncthreads();                                       // (the other buffer's readers passed the barrier of the tile before)
        if (kt + 1 < kt1) {
            sk.fetch(K, (kt + 1) * KT, klen, nch, tid);
            sv.fetch(V, (kt + 1) * KT, klen, nch, tid);
        }
        f32x16 s[MB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
            for (int j = 0; j < 16; ++j) s[mb][j] = 0.f;
#pragma unroll
            for (int kd = 0; kd < TL::NF; ++kd) s[mb] = TL::mma(TL::by_row(tk, mb * 32, kd, lane), qf[kd], s[mb]);
        }
        if (kt * KT + KT - 1 > lim0) {                         // a key of this tile is hidden from some row
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (kt * KT + mb * 32 + 8 * (j >> 2) + 4 * half + (j & 3) > lim) s[mb][j] = -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, s[mb][j]);
        top = half_swap_max(top) * c;
        const float mn = fmaxf(m, top), mu = mn == -__builtin_inff() ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - mu);
        m = mn;
        float sum = 0.f;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                s[mb][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mb][j], c, -mu));
                sum += s[mb][j];
            }
        l = __builtin_fmaf(l, alpha, sum);
        if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
            for (int i = 0; i < TL::DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= alpha;
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int kf = 0; kf < TL::CF; ++kf) {
                const u32x4 pf = TL::from_acc(s[mb], kf);
#pragma unroll
                for (int i = 0; i < TL::DB; ++i) o[i] = TL::mma(TL::by_col(tv, mb * 32, i, kf, lane), pf, o[i]);
            }
    }
    l = lim < 0 ? 0.f : half_swap_sum(l);                      // (a row that sees nothing may have gone through tiles that its neighbours see)
    if (l == 0.f) {
        m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < TL::DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    }

    const int whole = d.Tq * d.G;                              // rows of the result: those behind the sequence's end are zeros
    if (row >= whole) return;
    if (a.nsplit > 1) {
        const long at = ((long)split * d.nbh + bh) * whole + row;
        float* ml = a.part + (long)a.nsplit * d.nbh * whole * DP + at * 2;
        if (half == 0) { ml[0] = m; ml[1] = l; }
        if (l == 0.f) return;                                  // (nothing seen: the join takes no O from here)
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
    T* po = (T*)a.out + (((long)b * d.Tq + tok) * d.H + h) * d.D;
#pragma unroll
    for (int i = 0; i < TL::DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = i * 32 + g * 8 + half * 4;
            if (e < d.D) store4<T>(po + e, o[i][4 * g] * inv, o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv);
        }
    if (a.lse && half == 0)
        a.lse[((long)b * d.H + h) * d.Tq + tok] = l == 0.f ? -__builtin_inff() : m + __builtin_amdgcn_logf(l);
}

// joins the splits of a row: O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s; a wave per row
template <class T, int DP> __global__ __launch_bounds__(256) void attn_join_kernel(const AttnFwd a) {
    const AttnDims& d = a.d;
    const int whole = d.Tq * d.G, lane = threadIdx.x & 63;
    const long n = (long)d.nbh * whole, at = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= n) return;
    const float* ml = a.part + (long)a.nsplit * n * DP;
    float m = -__builtin_inff();
    for (int s = 0; s < a.nsplit; ++s) m = fmaxf(m, ml[(s * n + at) * 2]);
    const float mu = m == -__builtin_inff() ? 0.f : m;
    constexpr int E = DP >= 64 ? DP / 64 : 1;
    float o[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
        const float ls = ml[(s * n + at) * 2 + 1], w = __builtin_amdgcn_exp2f(ml[(s * n + at) * 2] - mu);
        if (ls == 0.f) continue;
        l = __builtin_fmaf(w, ls, l);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 64 * e < DP) o[e] = __builtin_fmaf(w, a.part[(s * n + at) * DP + lane + 64 * e], o[e]);
    }
    const int bh = (int)(at / whole), row = (int)(at - (long)bh * whole), b = bh / d.Hkv, tok = row / d.G;
    const int h = (bh - b * d.Hkv) * d.G + (row - tok * d.G);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* po = (T*)a.out + (((long)b * d.Tq + tok) * d.H + h) * d.D;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < d.D) po[lane + 64 * e] = from_f32<T>(o[e] * inv);
    if (a.lse && lane == 0) a.lse[((long)b * d.H + h) * d.Tq + tok] = l == 0.f ? -__builtin_inff() : m + __builtin_amdgcn_logf(l);
}

// rows a workgroup takes, keys a tile has, workgroups that share a row's keys
struct AttnPlan { int nw, kt, nsplit, ntile, dp; };
static AttnPlan attn_fwd_plan(int B, int Hkv, int G, int Tq, int Tk, int D, int es) {
    AttnPlan p;
    const long rows = (long)Tq * G;
    p.dp = D <= 32 ? 32 : D <= 64 ? 64 : 128;
    p.nw = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
    p.kt = p.nw == 1 || es == 4 ? 32 : 64;
    p.ntile = (int)((rows + p.nw * 32 - 1) / (p.nw * 32));
    // split where the tiles alone leave the chip idle: up to 2048 waves, at least two key tiles each, at most 128 ways (the join reads them all)
    const long base = (long)B * Hkv * p.ntile, want = 2048 / p.nw, ktiles = (Tk + p.kt - 1) / p.kt;
    long s = base >= want / 2 ? 1 : want / base;
    s = s > ktiles / 2 ? ktiles / 2 : s;
    p.nsplit = (int)(s < 1 ? 1 : s > 128 ? 128 : s);
    return p;
}

template <class T, int DP> static int attn_fwd_t(const AttnFwd& a, const AttnPlan& p, hipStream_t stream) {
    const dim3 grid(attn_grid(a.d, p.ntile), p.nsplit);
    constexpr int KT = sizeof(T) == 4 ? 32 : 64;
    if (p.nw == 1) attn_fwd_kernel<T, DP, 1, 32><<<grid, 64, 0, stream>>>(a);
    else if (p.nw == 2) attn_fwd_kernel<T, DP, 2, KT><<<grid, 128, 0, stream>>>(a);
    else attn_fwd_kernel<T, DP, 4, KT><<<grid, 256, 0, stream>>>(a);
    if (p.nsplit > 1) {
        const long n = (long)a.d.nbh * a.d.Tq * a.d.G;
        attn_join_kernel<T, DP><<<(unsigned)((n + 3) / 4), 256, 0, stream>>>(a);
    }
    return ppv_last_error();
}
template <class T> static int attn_fwd_dp(const AttnFwd& a, const AttnPlan& p, hipStream_t stream) {
    return p.dp == 32 ? attn_fwd_t<T, 32>(a, p, stream) : p.dp == 64 ? attn_fwd_t<T, 64>(a, p, stream) : attn_fwd_t<T, 128>(a, p, stream);
}

// the checks that both directions share; 0 or an error
int attn_check(const PpvAttention* x, AttnDims* d) {
    const int es = x->dtype == 0 ? 4 : 2, v = 16 / es;
    if (!x->q || !x->k || !x->v || !x->out) return PPV_ERR_NULL;
    if (x->dtype < 0 || x->dtype > 2 || x->B < 1 || x->H < 1 || x->Hkv < 1 || x->H % x->Hkv || x->Tq < 1 || x->Tk < 0 || x->D < 1 || x->D > 128 ||
        x->D % v || !(x->scale > 0.f) || x->scale > 1e30f)
        return PPV_ERR_BAD_SIZE;
    if ((long)x->Tq * (x->H / x->Hkv) > 0x3fffffffL || x->Tk > 0x3fffffff || (long)x->B * x->Hkv > 0x3fffffffL) return PPV_ERR_BAD_SIZE;
    const long st[] = {x->sqb, x->sqt, x->sqh, x->skb, x->skt, x->skh, x->svb, x->svt, x->svh};
    for (long s : st)
        if (s < 0 || s % v) return PPV_ERR_BAD_SIZE;
    const void* ps[] = {x->q, x->k, x->v, x->out};
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
    return p.nsplit > 1 ? (size_t)p.nsplit * B * H * Tq * (p.dp + 2) * sizeof(float) : 0;
}

int ppv_attention_fwd(const PpvAttention* x, ppv_stream_t stream) {
    if (!x) return PPV_ERR_NULL;
    AttnFwd a = {};
    if (int e = attn_check(x, &a.d)) return e;
    const AttnPlan p = attn_fwd_plan(x->B, x->Hkv, a.d.G, x->Tq, x->Tk, x->D, x->dtype == 0 ? 4 : 2);
    if (p.nsplit > 1 && !x->workspace) return PPV_ERR_WORKSPACE;
    if ((size_t)a.d.nbh * p.ntile > 0x7ffffff0u) return PPV_ERR_BAD_SIZE;
    a.q = {x->q, x->sqb, x->sqt, x->sqh};
    a.k = {x->k, x->skb, x->skt, x->skh};
    a.v = {x->v, x->svb, x->svt, x->svh};
    a.out = x->out;
    a.lse = x->lse;
    a.part = (float*)x->workspace;
    a.nsplit = p.nsplit;
    a.ntile = p.ntile;
    return x->dtype == 0 ? attn_fwd_dp<float>(a, p, stream) : x->dtype == 1 ? attn_fwd_dp<bf16s>(a, p, stream) : attn_fwd_dp<f16s>(a, p, stream);
}

}  // extern "C"
