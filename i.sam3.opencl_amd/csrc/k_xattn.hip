/* SPDX-License-Identifier: Unlicense
 *
 * Cross attention to another sequence's keys and values (cross_attend).
 *
 * Per (batch b, key head g) unit the queries of the heads that share the
 * key head are rows of one problem: row r is query r % n of head r / n of the
 * group, n the batch's queries, so that shared heads read K and V once.
 * o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j, in one
 * pass over the keys with the running maximum m and sum.
 *
 * A wave owns 32 rows and forms S^T = K Q^T and O^T = V^T P^T on 32 x 32
 * MFMA tiles: a lane then holds one row (column of S^T), row statistics need
 * one exchange with the lane 32 away, and the accumulator registers of S^T
 * are P's operand of the second product as they stand: contraction step s of
 * half h takes keys 16 s + 4 h + {0..3, 8..11}, and V is read in that order.
 * Halves and bfloat16 take v_mfma_f32_32x32x16, V transposed on its way out of
 * LDS (ds_read_b64_tr_b16); floats take v_mfma_f32_32x32x2, so that their
 * products are float products.
 *
 * Tiles of TK keys pass from memory through registers (loaded a tile ahead)
 * into LDS rows padded by 16 bytes, which leaves neither the 16-byte row reads
 * nor the transposed ones a bank conflict. Keys past the length and masked
 * keys enter LDS as zeros and their scores as minus infinity, so nothing that
 * stands in their memory reaches a result.
 */
#include "k_common.h"

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

#define NEG_INF (-__builtin_inff())
/* A row's maximum moves (and its sums are rescaled) when a score passes it
 * by more than this, in powers of two: P stays below 2^8, exact in range for
 * halves, and most tiles rescale nothing. */
#define LAZY 8.0f

template <int DT> struct xt {
    static constexpr int size = 2;
    typedef uint16_t elem;
};
template <> struct xt<DT_F32> {
    static constexpr int size = 4;
    typedef float elem;
};

template <int DT> __device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if (DT == DT_BF16)
        return pack_bf16x2(lo, hi);
    f16x2 p;

    p.x = (_Float16)lo;
    p.y = (_Float16)hi;
    return __builtin_bit_cast(uint32_t, p);
}

template <int DT>
__device__ __forceinline__ f32x16 mfma16(u32x4 a, u32x4 b, f32x16 c)
{
    if (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

/* Four keys (rows of lds, 8 bytes per lane) of 16 columns, transposed: lane i
 * of a group of 16 gets column i of the rows that lanes 4 k .. 4 k + 3 name. */
__device__ __forceinline__ u32x2 lds_tr(const char *lds)
{
    return __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) i16x4 *)lds));
}

/* Value of the lane 32 away, combined by the caller: (lower half's, upper
 * half's) value of both halves. */
__device__ __forceinline__ f32x2 both_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                    __builtin_bit_cast(uint32_t, v), false, false);
    f32x2 o;

    o.x = __builtin_bit_cast(float, (uint32_t)r[0]);
    o.y = __builtin_bit_cast(float, (uint32_t)r[1]);
    return o;
}

/* 16 bytes of a row at column byte cb: whole where vec, else element by
 * element, with zeros from column hd on. */
template <int DT>
__device__ __forceinline__ u32x4 row16(const char *p, int cb, int hdb, int vec)
{
    constexpr int S = xt<DT>::size;
    u32x4 v = {0, 0, 0, 0};

    if (cb >= hdb)
        return v;
    if (vec)
        return *(const u32x4 *)(p + cb);
    if (S == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (cb + 4 * i < hdb)
                v[i] = *(const uint32_t *)(p + cb + 4 * i);
    }
    else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (cb + 2 * i < hdb)
                v[i / 2] |= (uint32_t) * (const uint16_t *)(p + cb + 2 * i) << (16 * (i & 1));
    }
    return v;
}

/* Four consecutive columns from c of output row p (S bytes each), c < hd. */
template <int DT>
__device__ __forceinline__ void put_elem(char *p, int c, float v)
{
    if (DT == DT_F32)
        ((float *)p)[c] = v;
    else if (DT == DT_BF16)
        ((uint16_t *)p)[c] = f2bf(v);
    else
        ((_Float16 *)p)[c] = (_Float16)v;
}

/* DP: head width padded to 32, 64, 128 or 256. WM waves share the rows of a
 * workgroup, 4 / WM the keys of a tile. TK: keys of a tile. */
template <int DT, int DP, int WM, int TK>
__global__ __launch_bounds__(256, DP == 256 || (DP == 128 && DT == DT_F32 && WM < 4) ? 1 : 2) void k_xattn(const struct xattn_desc a)
{
    constexpr int S = xt<DT>::size;
    constexpr int WK = 4 / WM;
    constexpr int KW = TK / WK;          /* keys of a tile that a wave takes */
    constexpr int NB = KW / 32;          /* 32-key blocks of them */
    constexpr int CH = DP * S / 16;      /* 16-byte chunks of a row */
    constexpr int PITCH = DP * S + 16;
    constexpr int NL = TK * CH / 256;    /* chunks per thread, K or V */
    constexpr int MERGE = WK > 1 ? 4 * 32 * (DP + 4) * 4 + 4 * 32 * 8 : 0;
    constexpr int TILES = 2 * TK * PITCH;
    __shared__ __attribute__((aligned(16))) char lds[TILES > MERGE ? TILES : MERGE];
    char *const ldk = lds, *const ldv = lds + TK * PITCH;

    static_assert(NL * 256 == TK * CH && KW % 32 == 0 && TK <= 128, "tile");
    const int tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = l >> 5, lr = l & 31;
    const int wm = w % WM, wk = w / WM;

    /* Work item: XCD x (workgroup index mod 8) takes a contiguous range, so
     * that neighbours share its L2. */
    const long per = (a.items + 7) / 8;
    const long item = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);

    if (item >= a.items || (long)(blockIdx.x >> 3) >= per)
        return;
    int split, tile, unit;

    if (a.heads_first) {
        unit = (int)(item % a.units);
        tile = (int)(item / a.units % a.tiles);
        split = (int)(item / a.units / a.tiles);
    }
    else {
        tile = (int)(item % a.tiles);
        split = (int)(item / a.tiles % a.splits);
        unit = (int)(item / a.tiles / a.splits);
    }
    const int b = unit / a.kvh, kh = unit % a.kvh;
    const int nq = a.qlen ? max(0, min(a.qlen[b], a.Nq)) : a.Nq;
    const int nk = a.klen ? max(0, min(a.klen[b], a.Nk)) : a.Nk;
    const int rows = a.grp * nq;
    const int r0 = tile * WM * 32;

    if (r0 >= rows)
        return;
    const int per_split = ((nk + a.splits - 1) / a.splits + TK - 1) / TK * TK;
    const int jb = min(nk, split * per_split), je = min(nk, jb + per_split);
    const int hdb = a.hd * S;

    /* This lane's row: query and head, and its part of Q. */
    const int r = r0 + wm * 32 + lr;
    const int rc = min(r, rows - 1);
    const int hq = rc / nq, iq = rc % nq;
    const long orow = a.oo + (long)b * a.os0 + (long)(kh * a.grp + hq) * a.os1 + (long)iq * a.old;
    u32x4 qf[CH / 2];
    {
        const char *q = (const char *)a.Q +
                        S * (a.qo + (long)b * a.qs0 + (long)(kh * a.grp + hq) * a.qs1 +
                             (long)iq * a.qld);

#pragma unroll
        for (int i = 0; i < CH / 2; i++)
            qf[i] = row16<DT>(q, 16 * (2 * i + h), hdb, a.qvec);
    }
    const char *kb = (const char *)a.K + S * (a.ko + (long)b * a.ks0 + (long)kh * a.ks1);
    const char *vb = (const char *)a.V + S * (a.vo + (long)b * a.vs0 + (long)kh * a.vs1);
    const uint8_t *mk = a.kmask ? a.kmask + (long)b * a.Nk : nullptr;
    const uint32_t kstep = (uint32_t)a.kld * S, vstep = (uint32_t)a.vld * S;

    u32x4 sk[NL], sv[NL];
    auto load = [&](int j0) {
        const char *kt = kb + (long)j0 * kstep, *vt = vb + (long)j0 * vstep;
        const int last = je - 1 - j0;

#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int c = tid + 256 * i, row = c / CH, cb = c % CH * 16;
            const int rr = min(row, last);

            sk[i] = row16<DT>(kt + (uint32_t)rr * kstep, cb, hdb, a.kvec);
            sv[i] = row16<DT>(vt + (uint32_t)rr * vstep, cb, hdb, a.vvec);
        }
        if (mk || last < TK - 1) {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int row = (tid + 256 * i) / CH;
                const bool ok = row <= last && (!mk || mk[j0 + min(row, last)]);

                if (!ok)
                    sk[i] = sv[i] = u32x4{0, 0, 0, 0};
            }
        }
    };
    auto store = [&]() {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int c = tid + 256 * i, row = c / CH, cb = c % CH * 16;

            *(u32x4 *)(ldk + row * PITCH + cb) = sk[i];
            *(u32x4 *)(ldv + row * PITCH + cb) = sv[i];
        }
    };

    f32x16 o[DP / 32];
    float m = NEG_INF, sum = 0.0f;

#pragma unroll
    for (int i = 0; i < DP / 32; i++)
        o[i] = f32x16{0};
    if (jb < je)
        load(jb);
    for (int j0 = jb; j0 < je; j0 += TK) {
        __syncthreads();
        store();
        __syncthreads();
        /* Which of this wave's keys count, a bit for each. */
        uint64_t keep;
        {
            const int j = j0 + wk * KW + l;
            bool ok = l < KW && j < je;

            if (mk)
                ok = ok && mk[min(j, je - 1)] != 0;
            keep = __ballot(ok);
        }
        if (j0 + TK < je)
            load(j0 + TK);
        if (keep == 0)
            continue;
        f32x16 s[NB];

#pragma unroll
        for (int n = 0; n < NB; n++) {
            const char *kr = ldk + (wk * KW + n * 32 + lr) * PITCH + 16 * h;

            s[n] = f32x16{0};
#pragma unroll
            for (int i = 0; i < CH / 2; i++) {
                const u32x4 kf = *(const u32x4 *)(kr + 32 * i);

                if constexpr (DT == DT_F32) {
                    const f32x4 kx = __builtin_bit_cast(f32x4, kf);
                    const f32x4 qx = __builtin_bit_cast(f32x4, qf[i]);

#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(kx[e], qx[e], s[n], 0, 0, 0);
                }
                else
                    s[n] = mfma16<DT>(kf, qf[i], s[n]);
            }
        }
        if (KW == 64 ? ~keep != 0 : (uint32_t)keep != 0xffffffffu) {
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const uint32_t bits = (uint32_t)(keep >> (32 * n)) >> (4 * h);

#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!(bits >> (8 * (i / 4) + i % 4) & 1))
                        s[n][i] = NEG_INF;
            }
        }
        float mx = s[0][0];

#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 16; i++)
                mx = fmaxf(mx, s[n][i]);
        const f32x2 mh = both_halves(mx);

        mx = fmaxf(mh.x, mh.y) * a.c;
        if (__any(mx > m + LAZY)) {
            const float mn = fmaxf(m, mx);
            const float f = __builtin_amdgcn_exp2f(m - (mn == NEG_INF ? 0.0f : mn));

            m = mn;
            sum *= f;
#pragma unroll
            for (int d = 0; d < DP / 32; d++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    o[d][i] *= f;
        }
        const float ref = m == NEG_INF ? 0.0f : m;

#pragma unroll
        for (int n = 0; n < NB; n++) {
            float t[4] = {0, 0, 0, 0};

#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i], a.c, -ref));
                t[i & 3] += s[n][i];
            }
            sum += (t[0] + t[1]) + (t[2] + t[3]);
        }
#pragma unroll
        for (int n = 0; n < NB; n++) {
            if constexpr (DT == DT_F32) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const char *vr = ldv +
                                     (wk * KW + n * 32 + 8 * (i / 4) + i % 4 + 4 * h) * PITCH +
                                     4 * lr;

#pragma unroll
                    for (int d = 0; d < DP / 32; d++)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                            *(const float *)(vr + 128 * d), s[n][i], o[d], 0, 0, 0);
                }
            }
            else {
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    const char *vr = ldv +
                                     (wk * KW + n * 32 + 16 * st + 4 * h + (l & 15) / 4) * PITCH +
                                     32 * (l >> 4 & 1) + 8 * (l & 3);
                    u32x4 p;

#pragma unroll
                    for (int i = 0; i < 4; i++)
                        p[i] = pack2<DT>(s[n][8 * st + 2 * i], s[n][8 * st + 2 * i + 1]);
#pragma unroll
                    for (int d = 0; d < DP / 32; d++) {
                        const u32x2 v0 = lds_tr(vr + 64 * d), v1 = lds_tr(vr + 8 * PITCH + 64 * d);
                        const u32x4 vf = {v0.x, v0.y, v1.x, v1.y};

                        o[d] = mfma16<DT>(vf, p, o[d]);
                    }
                }
            }
        }
    }
    /* The two halves of a row's sum. */
    const f32x2 sh = both_halves(sum);

    sum = sh.x + sh.y;
    if (WK > 1) {
        /* The waves that share the rows: everything to the common maximum,
         * then added through LDS. */
        constexpr int OP = DP + 4;       /* floats of a row of partial sums */
        float *const po = (float *)lds + (long)(w * 32) * OP;
        float2 *const pm = (float2 *)(lds + 4 * 32 * OP * 4);

        __syncthreads();
        if (h == 0)
            pm[w * 32 + lr] = float2{m, sum};
        __syncthreads();
        float mm = m, ss = 0.0f;

#pragma unroll
        for (int k = 0; k < WK; k++)
            mm = fmaxf(mm, pm[(k * WM + wm) * 32 + lr].x);
        const float ref = mm == NEG_INF ? 0.0f : mm;

#pragma unroll
        for (int k = 0; k < WK; k++) {
            const float2 x = pm[(k * WM + wm) * 32 + lr];

            ss += x.y * __builtin_amdgcn_exp2f(x.x - ref);
        }
        const float f = __builtin_amdgcn_exp2f(m - ref);

#pragma unroll
        for (int d = 0; d < DP / 32; d++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                f32x4 t;

#pragma unroll
                for (int e = 0; e < 4; e++)
                    t[e] = o[d][4 * q + e] * f;
                *(f32x4 *)(po + lr * OP + 32 * d + 8 * q + 4 * h) = t;
            }
        __syncthreads();
        /* Wave w adds and keeps the d blocks wk, wk + WK, ... of its rows:
         * the registers it stores below. */
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
            if (d % WK == wk)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    f32x4 t = {0, 0, 0, 0};

#pragma unroll
                    for (int k = 0; k < WK; k++)
                        t += *(const f32x4 *)((float *)lds + ((k * WM + wm) * 32 + lr) * OP +
                                              32 * d + 8 * q + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[d][4 * q + e] = t[e];
                }
        m = mm;
        sum = ss;
    }
    if (r >= rows)
        return;
    if (a.splits > 1) {
        /* A record of this split: (m, sum) and the unnormalised sums. */
        const long ur = ((long)split * a.units + unit) * ((long)a.grp * a.Nq) + r;
        float *const rec = a.part + ur * a.hd;

        if (h == 0 && wk == 0)
            ((float2 *)(a.part + a.part_ml))[ur] = float2{m, sum};
        if (jb < je) {
#pragma unroll
            for (int d = 0; d < DP / 32; d++)
                if (d % WK == wk)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int c = 32 * d + 8 * q + 4 * h;

                        if (a.pvec) {
                            if (c < a.hd)
                                *(f32x4 *)(rec + c) = f32x4{o[d][4 * q], o[d][4 * q + 1],
                                                            o[d][4 * q + 2], o[d][4 * q + 3]};
                        }
                        else
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (c + e < a.hd)
                                    rec[c + e] = o[d][4 * q + e];
                    }
        }
        return;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    char *const op = (char *)a.O + S * orow;

#pragma unroll
    for (int d = 0; d < DP / 32; d++) {
        if (d % WK != wk)
            continue;
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            float x[8];

#pragma unroll
            for (int e = 0; e < 8; e++)
                x[e] = o[d][4 * q + e] * inv;
            const int c = 32 * d + 8 * q;

            if (!a.ovec) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int ce = c + 8 * (e / 4) + 4 * h + e % 4;

                    if (ce < a.hd)
                        put_elem<DT>(op, ce, x[e]);
                }
            }
            else if constexpr (DT == DT_F32) {
                if (c + 4 * h < a.hd)
                    *(f32x4 *)(op + 4 * (c + 4 * h)) = f32x4{x[0], x[1], x[2], x[3]};
                if (c + 8 + 4 * h < a.hd)
                    *(f32x4 *)(op + 4 * (c + 8 + 4 * h)) = f32x4{x[4], x[5], x[6], x[7]};
            }
            else {
                /* Lanes 32 apart exchange halves: 8 columns in a row each. */
                const auto u = __builtin_amdgcn_permlane32_swap(
                    pack2<DT>(x[0], x[1]), pack2<DT>(x[4], x[5]), false, false);
                const auto v = __builtin_amdgcn_permlane32_swap(
                    pack2<DT>(x[2], x[3]), pack2<DT>(x[6], x[7]), false, false);

                if (c + 8 * h < a.hd)
                    *(u32x4 *)(op + 2 * (c + 8 * h)) =
                        u32x4{(uint32_t)u[0], (uint32_t)v[0], (uint32_t)u[1], (uint32_t)v[1]};
            }
        }
    }
}

/* The splits of a row, a wave each: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s -
 * M) l_s with M the largest m_s. */
template <int DT>
__global__ __launch_bounds__(256) void k_xattn_merge(const struct xattn_desc a)
{
    const long ur = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long nrow = (long)a.grp * a.Nq, total = nrow * a.units;
    const int l = threadIdx.x & 63;

    if (ur >= total)
        return;
    const int unit = (int)(ur / nrow), r = (int)(ur % nrow);
    const int b = unit / a.kvh, kh = unit % a.kvh;
    const int nq = a.qlen ? max(0, min(a.qlen[b], a.Nq)) : a.Nq;

    if (r >= a.grp * nq)
        return;
    const float2 *ml = (const float2 *)(a.part + a.part_ml) + ur;
    float m = NEG_INF, sum = 0.0f;

    for (int s = 0; s < a.splits; s++)
        m = fmaxf(m, ml[s * total].x);
    const float ref = m == NEG_INF ? 0.0f : m;

    for (int s = 0; s < a.splits; s++)
        sum += ml[s * total].y * __builtin_amdgcn_exp2f(ml[s * total].x - ref);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    char *const op = (char *)a.O +
                     (long)xt<DT>::size * (a.oo + (long)b * a.os0 +
                                           (long)(kh * a.grp + r / nq) * a.os1 +
                                           (long)(r % nq) * a.old);

    for (int c = l; c < a.hd; c += 64) {
        float o = 0.0f;

        for (int s = 0; s < a.splits; s++) {
            const float2 x = ml[s * total];

            /* A split without keys left no sums. */
            if (x.y != 0.0f)
                o += a.part[(ur + s * total) * a.hd + c] * __builtin_amdgcn_exp2f(x.x - ref);
        }
        put_elem<DT>(op, c, o * inv);
    }
}

/* ------------------------------------------------------------ launch */

/* Head widths are padded to 32, 64, 128 or 256. */
static int padded(int hd)
{
    return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
}

/* Rows of 32 of a workgroup (the rest of its four waves split the keys) and
 * the key splits. Sets wm and splits of the problem. */
static void plan(struct xattn_desc *d)
{
    const int cu = dev_cu_count();
    const long rows = (long)d->grp * d->Nq;
    long wg;
    int wm = rows > 64 ? 4 : rows > 32 ? 2 : 1;

    if (wm == 1 && d->dt == DT_F32 && padded(d->hd) == 256)
        wm = 2;
    while (wm > 1 && !(wm == 2 && d->dt == DT_F32 && padded(d->hd) == 256) &&
           (long)d->units * ((rows + 32 * wm - 1) / (32 * wm)) < cu && d->Nk > 64 * 4 / wm)
        wm /= 2;
    d->wm = wm;
    d->tiles = (int)((rows + 32 * wm - 1) / (32 * wm));
    wg = (long)d->units * d->tiles;
    d->splits = 1;
    if (wg < 2 * cu) {
        const long most = d->Nk / (wm == 1 ? 256 : 128);

        d->splits = (int)((2 * cu + wg - 1) / wg);
        if (d->splits > most)
            d->splits = (int)most;
        if (d->splits > 64)
            d->splits = 64;
        if (d->splits < 1)
            d->splits = 1;
    }
    d->items = wg * d->splits;
    d->heads_first = d->Nk <= 256;
}

/* Offset of the splits' (m, sum) pairs in floats, and all of the workspace
 * in bytes. */
static size_t part_ml(const struct xattn_desc *d)
{
    return ((size_t)d->splits * d->units * d->grp * d->Nq * d->hd + 3) & ~(size_t)3;
}

extern "C" size_t xattn_ws(struct xattn_desc *d)
{
    plan(d);
    if (d->splits == 1)
        return 0;
    return 4 * part_ml(d) + 8 * (size_t)d->splits * d->units * d->grp * d->Nq;
}

template <int DT, int DP, int WM, int TK>
static int run(const struct xattn_desc *d, hipStream_t s)
{
    const long grid = (d->items + 7) / 8 * 8;

    hipLaunchKernelGGL((k_xattn<DT, DP, WM, TK>), dim3((unsigned)grid), dim3(256), 0, s, *d);
    return hipGetLastError();
}

template <int DT, int DP> static int run_wm(const struct xattn_desc *d, hipStream_t s)
{
    constexpr bool wide = DP * xt<DT>::size >= 512;

    if (d->wm == 4)
        return run<DT, DP, 4, wide ? 32 : 64>(d, s);
    if (d->wm == 2)
        return run<DT, DP, 2, 64>(d, s);
    if constexpr (DP * xt<DT>::size <= 512)
        return run<DT, DP, 1, 128>(d, s);
    return hipErrorInvalidValue;
}

template <int DT> static int run_dt(struct xattn_desc *d, hipStream_t s)
{
    const int dp = padded(d->hd);
    int err = dp == 32    ? run_wm<DT, 32>(d, s)
              : dp == 64  ? run_wm<DT, 64>(d, s)
              : dp == 128 ? run_wm<DT, 128>(d, s)
                          : run_wm<DT, 256>(d, s);

    if (err == hipSuccess && d->splits > 1) {
        const long rows = (long)d->units * d->grp * d->Nq;

        hipLaunchKernelGGL((k_xattn_merge<DT>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s,
                           *d);
        err = hipGetLastError();
    }
    return err;
}

extern "C" int launch_xattn(struct xattn_desc *d, void *ws, size_t ws_bytes, void *stream)
{
    const size_t need = xattn_ws(d);

    if (need && (!ws || ws_bytes < need)) {
        /* One workgroup per row tile walks all keys. */
        d->splits = 1;
        d->items = (long)d->units * d->tiles;
    }
    d->part = (float *)ws;
    d->part_ml = d->splits > 1 ? (long)part_ml(d) : 0;
    if (d->dt == DT_F32)
        return run_dt<DT_F32>(d, (hipStream_t)stream);
    if (d->dt == DT_F16)
        return run_dt<DT_F16>(d, (hipStream_t)stream);
    return run_dt<DT_BF16>(d, (hipStream_t)stream);
}
