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
 * Tiles of TK keys are copied straight into LDS (global_load_lds_dwordx4) a
 * tile or more ahead of their use, the 16-byte chunks of a row swizzled so that
 * neither the row reads of K nor the transposed reads of V meet a bank
 * conflict. Operands whose rows do not start on 16 bytes take the same path
 * through registers, element by element. Scores of keys past the length and
 * of masked ones become minus infinity and their rows of V zeros, so nothing
 * that stands in their memory reaches a result.
 */
#include "k_xattn.h"

/* DP: head width padded to 32, 64, 128 or 256, of which the first DB blocks of 32
 * hold columns. WM waves share the rows of a
 * workgroup, the rest of its four the keys of a tile; WM = 8 is eight waves, each
 * with rows of its own. TK: keys of a tile. ST: tiles in LDS, ST - 1 of them
 * ahead. VEC: the rows of all operands are whole 16-byte pieces. */
template <int DT, int DP, int DB, int WM, int TK, int ST, int OCC, bool VEC>
__global__ __launch_bounds__(WM == 8 ? 512 : 256, OCC) void k_xattn(const struct xattn_desc a)
{
    constexpr int S = xt<DT>::size;
    constexpr int NW = WM == 8 ? 8 : 4;
    constexpr int WK = NW / WM;
    constexpr int KW = TK / WK;          /* keys of a tile that a wave takes */
    constexpr int NB = KW / 32;          /* 32-key blocks of them */
    constexpr int RB = DP * S;           /* bytes of a row */
    constexpr int CH = RB / 16;          /* 16-byte chunks of a row */
    constexpr int QS = DB * S;           /* steps of 32 bytes of the first product */
    constexpr int NI = TK * RB / (1024 * NW); /* copies of a wave for K or V: 1 KiB each */
    constexpr int MERGE = WK > 1 ? 4 * 32 * (DP + 4) * 4 + 4 * 32 * 8 : 0;
    typedef row_k<RB> rk;
    typedef row_v<RB, DT> rv;
    constexpr int KT = TK / rk::RPK * (1024 + rk::PAD); /* LDS bytes of a tile's K */
    constexpr int TILE = KT + TK / rv::RPK * (1024 + rv::PAD);
    __shared__ __attribute__((aligned(1024))) char lds[ST * TILE > MERGE ? ST * TILE : MERGE];

    static_assert(NI >= 1 && KW % 32 == 0 && KW <= 64 && TK <= 128, "tile");
    const int tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = l >> 5, lr = l & 31;
    const int wm = w % WM, wk = w / WM;

    unsigned split, tile, unit;

    if (a.heads_first) {
        if (!item_of(a.tiles, a.units, &tile, &unit))
            return;
        split = 0;
    }
    else {
        unsigned group;

        if (!item_of(a.units * a.splits, a.tiles, &group, &tile))
            return;
        unit = group / a.splits;
        split = group - unit * a.splits;
    }
    const int b = unit / (unsigned)a.kvh, kh = unit - b * a.kvh;
    const int nq = a.qlen ? max(0, min(a.qlen[b], a.Nq)) : a.Nq;
    const int nk = a.klen ? max(0, min(a.klen[b], a.Nk)) : a.Nk;
    const int rows = a.grp * nq;
    const int r0 = tile * WM * 32;

    if (r0 >= rows)
        return;
    /* Every splits-th tile, so that splits have like shares of what a mask
     * leaves. */
    const int hop = TK * a.splits, jb = TK * split, je = nk;
    const int hdb = a.hd * S;

    const char *const kb = (const char *)a.K + S * (a.ko + (long)b * a.ks0 + (long)kh * a.ks1);
    const char *const vb = (const char *)a.V + S * (a.vo + (long)b * a.vs0 + (long)kh * a.vs1);
    const uint8_t *const mk = a.kmask ? a.kmask + (long)b * a.Nk : nullptr;
    const uint32_t kstep = (uint32_t)a.kld * S, vstep = (uint32_t)a.vld * S;

    /* Copy i of this wave fills rows (w NI + i) RPK on of a tile; lane l's 16
     * bytes are of row l / CH of them. koff, voff: their offsets in memory from
     * the copy's first row (columns of blocks that are not used stand for any:
     * the first ones). lk, lv: where the wave's copies go in slot 0. */
    const int lrow = l / CH;
    const int ck = 16 * ((l % CH) ^ rk::swz(lrow)), cv = 16 * ((l % CH) ^ rv::swz(lrow));
    const uint32_t koff = lrow * kstep + (ck < hdb ? ck : 0), voff = lrow * vstep + (cv < hdb ? cv : 0);
    const unsigned lk = (unsigned)(uintptr_t)lds + w * NI * (1024 + rk::PAD);
    const unsigned lv = (unsigned)(uintptr_t)lds + KT + w * NI * (1024 + rv::PAD);
    /* Starts the copies of a tile of which every row is whole, from rows kt and
     * vt (the wave's first) into slot st. */
    auto copy_full = [&](const char *kt, const char *vt, int st) {
        const unsigned tk = __builtin_amdgcn_readfirstlane(lk + st * TILE);
        const unsigned tv = __builtin_amdgcn_readfirstlane(lv + st * TILE);

#pragma unroll
        for (int i = 0; i < NI; i++) {
            g2lds16(kt + (long)(i * rk::RPK) * kstep, koff, tk + (1024 + rk::PAD) * i);
            g2lds16(vt + (long)(i * rv::RPK) * vstep, voff, tv + (1024 + rv::PAD) * i);
        }
    };
    /* The tile at key j0, up to key je (its last row stands for those behind)
     * and column hd (zeros behind). */
    auto copy = [&](int j0, int st) {
        const int last = je - 1 - j0, w0 = w * NI * rk::RPK;

        if (VEC && a.hd == 32 * DB && last >= TK - 1) {
            copy_full(kb + (long)(j0 + w0) * kstep, vb + (long)(j0 + w0) * vstep, st);
            return;
        }
        const unsigned tk = __builtin_amdgcn_readfirstlane(lk + st * TILE);
        const unsigned tv = __builtin_amdgcn_readfirstlane(lv + st * TILE);

#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int rr = j0 + min(w0 + i * rk::RPK + lrow, last);
            const char *pk = kb + (long)rr * kstep, *pv = vb + (long)rr * vstep;

            if (VEC) {
                g2lds16_at(ck < hdb ? pk + ck : (const char *)&xattn_zeros,
                           tk + (1024 + rk::PAD) * i);
                g2lds16_at(cv < hdb ? pv + cv : (const char *)&xattn_zeros,
                           tv + (1024 + rv::PAD) * i);
            }
            else {
                char *const at = lds + st * TILE + 16 * l;

                *(u32x4 *)(at + (w * NI + i) * (1024 + rk::PAD)) = row16<DT, VEC>(pk, ck, hdb);
                *(u32x4 *)(at + KT + (w * NI + i) * (1024 + rv::PAD)) =
                    row16<DT, VEC>(pv, cv, hdb);
            }
        }
    };

    /* This split's tiles t = 0 .. tiles - 1; the first one from t on of which a
     * long mask leaves a key, and which of this wave's keys of it. Lane l looks up
     * tile k0 + l (a bit per key, bits in words of 32), so that masks cost no
     * copies of empty tiles and no loads in the loop, which would wait for the
     * copies under way too. us with masks that keep an eighth to a half, looked
     * up and read tile by tile: one token of 16 heads over 8192 keys, batch 4 14.8
     * and 21.0; 2000 x 2000 17.0 and 26.1; but 500 x 200 9.4 and 8.6, 200 x 77 8.0
     * and 6.8. */
    const bool ahead_mask = mk && a.Nk > 512;
    const int tiles = jb < je ? (je - jb + hop - 1) / hop : 0;
    uint64_t kept = 0;
    int k0 = -64;
    uint32_t word[NB];
    auto next = [&](int t, uint64_t *keep) {
        if (!ahead_mask)
            return t;
        for (; t < tiles; t = k0 + 64) {
            if (t >= k0 + 64) {
                const int j = jb + min(t + l, tiles - 1) * hop;
                uint32_t any = 0;

#pragma unroll
                for (int i = 0; i < TK / 32; i++) {
                    uint32_t bits = 0;

#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        const int at = j + 32 * i + 4 * c, past = max(at + 4 - je, 0);
                        uint32_t x = 0;

                        if (je >= 4)
                            __builtin_memcpy(&x, mk + min(at, je - 4), 4);
                        else
                            for (int e = 0; e < je; e++)
                                x |= (uint32_t)mk[e] << (8 * (4 - je + e));
                        x = past < 4 ? x >> (8 * past) : 0;
                        /* A byte's top bit: it is not zero. The four together. */
                        x = ((((x & 0x7f7f7f7f) + 0x7f7f7f7f) | x) >> 7 & 0x01010101) * 0x10204080;
                        bits |= x >> 28 << (4 * c);
                    }
                    any |= bits;
                    if (i / NB == wk)
                        word[i % NB] = bits;
                }
                k0 = t;
                kept = __ballot(any != 0 && t + l < tiles);
            }
            const uint64_t left = kept >> (t - k0);

            if (left) {
                t += __builtin_ctzll(left);
                *keep = (uint32_t)__builtin_amdgcn_readlane(word[0], t - k0);
                if (NB == 2)
                    *keep |= (uint64_t)__builtin_amdgcn_readlane(word[NB - 1], t - k0) << 32;
                return t;
            }
        }
        return tiles;
    };
    /* The tiles in LDS and the one to copy next. */
    int q[ST];
    uint64_t kq[ST];

    /* The first tiles, on their way while Q is read. */
#pragma unroll
    for (int i = 0; i < ST; i++)
        q[i] = next(i ? q[i - 1] + 1 : 0, kq + i);
#pragma unroll
    for (int i = 0; i < ST - 1; i++)
        if (q[i] < tiles)
            copy(jb + q[i] * hop, i);
    /* This lane's row: query and head, and its part of Q. */
    const int r = r0 + wm * 32 + lr;
    const int rc = min(r, rows - 1);
    const int hq = a.grp == 1 ? 0 : rc / nq, iq = rc - hq * nq;
    u32x4 qf[QS];
    {
        const char *q = (const char *)a.Q +
                        S * (a.qo + (long)b * a.qs0 + (long)(kh * a.grp + hq) * a.qs1 +
                             (long)iq * a.qld);

#pragma unroll
        for (int i = 0; i < QS; i++)
            qf[i] = row16<DT, VEC>(q, 16 * (2 * i + h), hdb);
    }
    /* Q has arrived: left to its first use, the wait for it would stand inside
     * the loop and wait for the copies of the next tile there each time. */
#pragma unroll
    for (int i = 0; i < QS; i++)
        asm volatile("" : "+v"(qf[i]));
    f32x16 o[DB];
    float m = NEG_INF, sum = 0.0f;

#pragma unroll
    for (int i = 0; i < DB; i++)
        o[i] = f32x16{0};
    /* This wave's keys of the tile in slot st: all of them, or those whose
     * bit in keep is set. */
    auto attend_tile = [&](auto all, int st, uint64_t keep) {
        constexpr bool ALL = decltype(all)::value;
        char *const ldk = lds + st * TILE + wk * rk::at(KW);
        char *const ldv = lds + st * TILE + KT + wk * rv::at(KW);
        /* The second block of 32 keys is empty. */
        const bool half = !ALL && NB == 2 && keep >> 32 == 0;
        f32x16 s[NB];

#pragma unroll
        for (int n = 0; n < NB; n++)
            s[n] = f32x16{0};
        if (half) {
#pragma unroll
            for (int i = 0; i < QS; i++)
                s[0] = k_step<DT>(*(const u32x4 *)(ldk + rk::at(lr) + 16 * ((2 * i + h) ^ rk::swz(lr))),
                                  qf[i], s[0]);
        }
        else {
#pragma unroll
            for (int i = 0; i < QS; i++)
#pragma unroll
                for (int n = 0; n < NB; n++)
                    s[n] = k_step<DT>(*(const u32x4 *)(ldk + rk::at(n * 32) + rk::at(lr) +
                                                       16 * ((2 * i + h) ^ rk::swz(lr))),
                                      qf[i], s[n]);
        }
        if (!ALL && (KW == 64 ? ~keep != 0 : (uint32_t)keep != 0xffffffffu)) {
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const uint32_t bits = (uint32_t)(keep >> (32 * n)) >> (4 * h);

#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!(bits >> (8 * (i / 4) + i % 4) & 1))
                        s[n][i] = NEG_INF;
            }
            /* Their rows of V, by each wave that reads them. */
            for (int c = l; c < KW * CH; c += 64)
                if (!(keep >> (c / CH) & 1))
                    *(u32x4 *)(ldv + rv::at(c / CH) + 16 * (c % CH)) = u32x4{0, 0, 0, 0};
            wave_lds_order();
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
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    o[d][i] *= f;
        }
        const float ref = m == NEG_INF ? 0.0f : m;

#pragma unroll
        for (int n = 0; n < NB; n++) {
            float t[4];

#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i], a.c, -ref));
                t[i & 3] = i < 4 ? s[n][i] : t[i & 3] + s[n][i];
            }
            sum += (t[0] + t[1]) + (t[2] + t[3]);
        }
#pragma unroll
        for (int n = 0; n < NB; n++) {
            if (n && half)
                break;
            if constexpr (DT == DT_F32) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const char *vr =
                        ldv + rv::at(n * 32 + 8 * (i / 4)) + rv::at(i % 4 + 4 * h) + 4 * lr;

#pragma unroll
                    for (int d = 0; d < DB; d++)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                            *(const float *)(vr + 128 * d), s[n][i], o[d], 0, 0, 0);
                }
            }
            else {
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int row = 4 * h + (l & 15) / 4;
                    const char *vr = ldv + rv::at(n * 32 + 16 * hf) + rv::at(row) + 8 * (l & 1);
                    const int c0 = 2 * (l >> 4 & 1) + (l >> 1 & 1);
                    u32x4 p;

#pragma unroll
                    for (int i = 0; i < 4; i++)
                        p[i] = pack2<DT>(s[n][8 * hf + 2 * i], s[n][8 * hf + 2 * i + 1]);
#pragma unroll
                    for (int d = 0; d < DB; d++) {
                        const char *vd = vr + 16 * ((4 * d + c0) ^ rv::swz(row));
                        const u32x2 v0 = lds_tr(vd), v1 = lds_tr(vd + rv::at(8));
                        const u32x4 vf = {v0.x, v0.y, v1.x, v1.y};

                        o[d] = mfma16<DT>(vf, p, o[d]);
                    }
                }
            }
        }
    };
    int st = 0;

    /* Whole tiles whose copies ahead are whole tiles too: nothing to check. */
    if (VEC && a.hd == 32 * DB && !mk) {
        const long ahead = jb + (ST - 1) * hop + w * NI * rk::RPK;
        const char *kt = kb + ahead * kstep, *vt = vb + ahead * vstep;

        int t = 0;

        for (int j = jb + (ST - 1) * hop; j + TK <= je; j += hop, t++) {
            copies_and_barrier<(ST - 2) * 2 * NI>();
            copy_full(kt, vt, st == 0 ? ST - 1 : st - 1);
            kt += (long)hop * kstep;
            vt += (long)hop * vstep;
            attend_tile(yes{}, st, 0);
            st = st + 1 == ST ? 0 : st + 1;
        }
#pragma unroll
        for (int i = 0; i < ST; i++)
            q[i] = t + i;
    }
    while (q[0] < tiles) {
        const int j0 = jb + q[0] * hop;
        const bool drop = mk && !ahead_mask &&
                          mk[min(j0 + wk * KW + (l & (KW - 1)), je - 1)] == 0;

        /* This tile has landed, and the slot of the one before is free. */
        if (ST > 2 && q[ST - 2] < tiles)
            copies_and_barrier<(ST - 2) * 2 * NI>();
        else
            copies_and_barrier<0>();
        if (q[ST - 1] < tiles)
            copy(jb + q[ST - 1] * hop, st == 0 ? ST - 1 : st - 1);
        /* Which of this wave's keys count. */
        const uint64_t keep =
            ahead_mask ? kq[0] : __ballot(l < KW && j0 + wk * KW + l < je && !drop);

        if (keep)
            attend_tile(no{}, st, keep);
#pragma unroll
        for (int i = 0; i < ST - 1; i++) {
            q[i] = q[i + 1];
            kq[i] = kq[i + 1];
        }
        q[ST - 1] = next(q[ST - 1] + 1, kq + ST - 1);
        st = st + 1 == ST ? 0 : st + 1;
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
        for (int d = 0; d < DB; d++)
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
        for (int d = 0; d < DB; d++)
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
            for (int d = 0; d < DB; d++)
                if (d % WK == wk)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int c = 32 * d + 8 * q + 4 * h;

                        if (VEC) {
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
    char *const op = (char *)a.O + S * (a.oo + (long)b * a.os0 + (long)(kh * a.grp + hq) * a.os1 +
                                        (long)iq * a.old);

#pragma unroll
    for (int d = 0; d < DB; d++)
        if (d % WK == wk)
            put_block<DT, VEC>(op, 32 * d, a.hd, h, o[d], inv);
}

/* At most 64 keys (a prompt) and many rows: bound by reading Q and writing O. A
 * workgroup keeps one unit's K and V and each of its waves walks blocks of 32
 * rows, the next block's rows of Q under way; all weights of a row are there at
 * once, so no maximum runs. Fragments of K and V stay in registers where the
 * types are 16 bits wide. us at batch 8, 5184 rows, 37 keys, 8 heads of 32 and 64
 * bf16 (43 and 85 MB): 12.3 and 21.2 (3.5 and 4.0 TB/s), 13.5 and 24.7 with a
 * lane per row of Q and O in memory, 16.6 and 24.6 by k_xattn; 13.4 for the first
 * with O through the caches, 14.7 with two blocks ahead, 17.1 with 8 instead of 4
 * workgroups per compute unit. Floats, 20 keys, heads of 32: 25.2, 30.2 by
 * k_xattn. */
template <int DT, int DP, int NB>
__global__ __launch_bounds__(256, 2) void k_xattn_few(const struct xattn_desc a)
{
    constexpr int S = xt<DT>::size;
    constexpr int RB = DP * S, CH = RB / 16;
    typedef row_k<RB> rk;
    typedef row_v<RB, DT> rv;
    constexpr int NK = NB * 32 / rk::RPK;               /* copies for K or V, 1 KiB each */
    constexpr int KT = NK * (1024 + rk::PAD);
    constexpr int NV = DT == DT_F32 ? 0 : 2 * NB * (DP / 32);
    constexpr int QP = RB + 16;                         /* pitch of a wave's own rows */
    constexpr int KV = KT + NK * (1024 + rv::PAD);
    __shared__ __attribute__((aligned(1024))) char lds[KV + 4 * 32 * QP];
    const int tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = l >> 5, lr = l & 31;
    char *const own = lds + KV + w * 32 * QP;
    unsigned part, unit;

    if (!item_of(a.tiles, a.units, &part, &unit))
        return;
    const int b = unit / (unsigned)a.kvh, kh = unit - b * a.kvh;
    const int nq = a.qlen ? max(0, min(a.qlen[b], a.Nq)) : a.Nq;
    const int nk = a.klen ? max(0, min(a.klen[b], a.Nk)) : a.Nk;
    const int rows = a.grp * nq, blocks = (rows + 31) / 32, hdb = a.hd * S;
    /* This wave's blocks: part, part + parts, ... of four waves each. */
    const int step = 4 * a.tiles;
    int blk = 4 * part + w;

    if (4 * (int)part >= blocks)
        return;
    /* Rows of Q and O pass through LDS of the wave's own: in memory CH lanes take
     * a whole row (a lane of each row at a time would be 64 requests). Access i
     * of lane l: row i 64 / CH + l / CH, 16 bytes l % CH. */
    auto row_at = [&](int blk, int i, long off, long s0, long s1, int ld) {
        const int r = min(blk * 32 + i * (64 / CH) + l / CH, rows - 1);
        const int hq = a.grp == 1 ? 0 : r / nq, iq = r - hq * nq;

        return S * (off + (long)b * s0 + (long)(kh * a.grp + hq) * s1 + (long)iq * ld) +
               16 * (l % CH);
    };
    u32x4 q[CH / 2];
    auto load_q = [&](int blk) {
#pragma unroll
        for (int i = 0; i < CH / 2; i++)
            q[i] = 16 * (l % CH) < hdb
                       ? *(const u32x4 *)((const char *)a.Q + row_at(min(blk, blocks - 1), i, a.qo,
                                                                     a.qs0, a.qs1, a.qld))
                       : u32x4{0, 0, 0, 0};
    };
    /* K and V: rows past the last key read the last one, columns past hd zeros. */
    const unsigned lbase = (unsigned)(uintptr_t)lds;

    if (nk > 0) {
        const int lrow = l / CH;
        const int ck = 16 * ((l % CH) ^ rk::swz(lrow)), cv = 16 * ((l % CH) ^ rv::swz(lrow));
        const char *const kb =
            (const char *)a.K + S * (a.ko + (long)b * a.ks0 + (long)kh * a.ks1);
        const char *const vb =
            (const char *)a.V + S * (a.vo + (long)b * a.vs0 + (long)kh * a.vs1);

        for (int c = w; c < NK; c += 4) {
            const long r = min(c * rk::RPK + lrow, nk - 1);

            g2lds16_at(ck < hdb ? kb + r * a.kld * S + ck : (const char *)&xattn_zeros,
                       __builtin_amdgcn_readfirstlane(lbase + c * (1024 + rk::PAD)));
            g2lds16_at(cv < hdb ? vb + r * a.vld * S + cv : (const char *)&xattn_zeros,
                       __builtin_amdgcn_readfirstlane(lbase + KT + c * (1024 + rv::PAD)));
        }
    }
    /* Keys that count, a bit for each. */
    const bool in = l < NB * 32 && l < nk;
    const uint64_t keep = __ballot(in && (!a.kmask || a.kmask[(long)b * a.Nk + min(l, nk - 1)]));

    load_q(blk);
    copies_and_barrier<0>();
    /* Rows of V that do not count. */
    for (int c = tid; c < NB * 32 * CH; c += 256)
        if (!(keep >> (c / CH) & 1))
            *(u32x4 *)(lds + KT + rv::at(c / CH) + 16 * (c % CH)) = u32x4{0, 0, 0, 0};
    copies_and_barrier<0>();
    auto k_frag = [&](int n, int i) {
        return *(const u32x4 *)(lds + rk::at(n * 32) + rk::at(lr) +
                                16 * ((2 * i + h) ^ rk::swz(lr)));
    };
    auto v_frag = [&](int f) {
        const int key = f / (DP / 32) * 16, d = f % (DP / 32);
        const int row = 4 * h + (l & 15) / 4, c0 = 2 * (l >> 4 & 1) + (l >> 1 & 1);
        const char *vd = lds + KT + rv::at(key) + rv::at(row) + 8 * (l & 1) +
                         16 * ((4 * d + c0) ^ rv::swz(row));
        const u32x2 v0 = lds_tr(vd), v1 = lds_tr(vd + rv::at(8));

        return u32x4{v0.x, v0.y, v1.x, v1.y};
    };
    u32x4 kf[NB * (CH / 2)], vf[NV + 1];

    if constexpr (DT != DT_F32) {
#pragma unroll
        for (int f = 0; f < NB * (CH / 2); f++)
            kf[f] = k_frag(f % NB, f / NB);
#pragma unroll
        for (int f = 0; f < NV; f++)
            vf[f] = v_frag(f);
    }
    for (; blk < blocks; blk += step) {
        f32x16 s[NB], o[DP / 32];
        float mx = NEG_INF, sum = 0.0f;

#pragma unroll
        for (int i = 0; i < CH / 2; i++)
            *(u32x4 *)(own + (i * (64 / CH) + l / CH) * QP + 16 * (l % CH)) = q[i];
        wave_lds_order();
        load_q(blk + step);
#pragma unroll
        for (int n = 0; n < NB; n++)
            s[n] = f32x16{0};
#pragma unroll
        for (int i = 0; i < CH / 2; i++) {
            const u32x4 qf = *(const u32x4 *)(own + lr * QP + 16 * (2 * i + h));

#pragma unroll
            for (int n = 0; n < NB; n++)
                s[n] = k_step<DT>(DT == DT_F32 ? k_frag(n, i) : kf[i * NB + n], qf, s[n]);
        }
        if (NB == 2 ? ~keep != 0 : (uint32_t)keep != 0xffffffffu)
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const uint32_t bits = (uint32_t)(keep >> (32 * n)) >> (4 * h);

#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!(bits >> (8 * (i / 4) + i % 4) & 1))
                        s[n][i] = NEG_INF;
            }
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 16; i++)
                mx = fmaxf(mx, s[n][i]);
        const f32x2 mh = both_halves(mx);

        mx = fmaxf(mh.x, mh.y) * a.c;
        mx = mx == NEG_INF ? 0.0f : mx;
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i], a.c, -mx));
                sum += s[n][i];
            }
        const f32x2 sh = both_halves(sum);

        sum = sh.x + sh.y;
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
            o[d] = f32x16{0};
        if constexpr (DT == DT_F32) {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const char *vr = lds + KT + rv::at(n * 32 + 8 * (i / 4)) +
                                     rv::at(i % 4 + 4 * h) + 4 * lr;

#pragma unroll
                    for (int d = 0; d < DP / 32; d++)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(*(const float *)(vr + 128 * d),
                                                                    s[n][i], o[d], 0, 0, 0);
                }
        }
        else {
#pragma unroll
            for (int k = 0; k < 2 * NB; k++) {
                u32x4 p;

#pragma unroll
                for (int i = 0; i < 4; i++)
                    p[i] = pack2<DT>(s[k / 2][8 * (k & 1) + 2 * i],
                                     s[k / 2][8 * (k & 1) + 2 * i + 1]);
#pragma unroll
                for (int d = 0; d < DP / 32; d++)
                    o[d] = mfma16<DT>(vf[k * (DP / 32) + d], p, o[d]);
            }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;

#pragma unroll
        for (int d = 0; d < DP / 32; d++)
            put_block<DT, true>(own + lr * QP, 32 * d, DP, h, o[d], inv);
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < CH / 2; i++) {
            const int r = i * (64 / CH) + l / CH;
            const u32x4 v = *(const u32x4 *)(own + r * QP + 16 * (l % CH));

            if (blk * 32 + r < rows && 16 * (l % CH) < hdb)
                __builtin_nontemporal_store(
                    v, (u32x4 *)((char *)a.O + row_at(blk, i, a.oo, a.os0, a.os1, a.old)));
        }
        wave_lds_order();
    }
}

/* The splits of a row: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, M the
 * largest m_s. LP lanes per row, four columns each (or one where rows are no
 * multiple of four), eight splits' loads under way at a time. */
template <int DT, int LP, bool VEC>
__global__ __launch_bounds__(256) void k_xattn_merge(const struct xattn_desc a)
{
    constexpr int V = VEC ? 4 : 1;
    const int lane = threadIdx.x % LP;
    const long ur = (long)blockIdx.x * (256 / LP) + threadIdx.x / LP;
    const long nrow = (long)a.grp * a.Nq, total = nrow * a.units;

    if (ur >= total)
        return;
    const int unit = (int)(ur / nrow), r = (int)(ur - unit * nrow);
    const int b = unit / a.kvh, kh = unit % a.kvh;
    const int nq = a.qlen ? max(0, min(a.qlen[b], a.Nq)) : a.Nq;

    if (r >= a.grp * nq)
        return;
    const float2 *ml = (const float2 *)(a.part + a.part_ml) + ur;
    char *const op = (char *)a.O +
                     (long)xt<DT>::size * (a.oo + (long)b * a.os0 +
                                           (long)(kh * a.grp + r / nq) * a.os1 +
                                           (long)(r % nq) * a.old);

    for (int c = lane * V; c < a.hd; c += LP * V) {
        const float *const rec = a.part + ur * a.hd + c;
        float m = NEG_INF, sum = 0.0f, o[V] = {0};

        for (int s0 = 0; s0 < a.splits; s0 += 8) {
            float2 x[8];
            float v[8][V];
            float mn = m;

#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int s = min(s0 + k, a.splits - 1);

                x[k] = ml[s * total];
                if constexpr (VEC)
                    *(f32x4 *)v[k] = *(const f32x4 *)(rec + s * total * a.hd);
                else
                    v[k][0] = rec[s * total * a.hd];
            }
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (s0 + k < a.splits)
                    mn = fmaxf(mn, x[k].x);
            const float ref = mn == NEG_INF ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - ref);

            m = mn;
            sum *= f;
#pragma unroll
            for (int e = 0; e < V; e++)
                o[e] *= f;
#pragma unroll
            for (int k = 0; k < 8; k++)
                /* A split without keys left no sums. */
                if (s0 + k < a.splits && x[k].y != 0.0f) {
                    const float g = __builtin_amdgcn_exp2f(x[k].x - ref);

                    sum = fmaf(g, x[k].y, sum);
#pragma unroll
                    for (int e = 0; e < V; e++)
                        o[e] = fmaf(g, v[k][e], o[e]);
                }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;

#pragma unroll
        for (int e = 0; e < V; e++)
            o[e] *= inv;
        if constexpr (!VEC)
            put_elem<DT>(op, c, o[0]);
        else if constexpr (DT == DT_F32)
            *(f32x4 *)(op + 4 * c) = f32x4{o[0], o[1], o[2], o[3]};
        else
            *(u32x2 *)(op + 2 * c) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
    }
}

/* ------------------------------------------------------------ launch */

/* Head widths are padded to 32, 64, 128 or 256. */
static int padded(int hd)
{
    return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
}

/* Time of floats in f32 plans, in 32 rows x one key on a SIMD, wm waves' rows in
 * s splits: the compute unit with most workgroups, their start (and, with the
 * keys in four waves, the copies, which bind: 1.2), the merge's launch and the
 * splits' records. */
static double cost_f32(const struct xattn_desc *d, int wm, int s, long rows, long cu)
{
    const long wg = d->units * ((rows + 32 * wm - 1) / (32 * wm)) * s;
    const double keys = ((d->Nk + s - 1) / s + 63) / 64 * 64.0, rounds = (wg + cu - 1) / cu;
    const double c = rounds * (wm == 1 ? 1.2 * (keys + 128) : wm * (keys + 64));

    return s == 1 ? c : c + 12000.0 / padded(d->hd) + 0.005 * d->units * rows * s;
}

/* How the work is cut. A workgroup of wm x 32 rows walks all keys of its rows,
 * or one of several splits of them whose sums a second launch adds up. More rows
 * share each copied tile; fewer make more workgroups, whose waves then share
 * the keys. us on 256 compute units, f16 but for the last, wm 4 / 2 / 1:
 *   12 heads of 64, 447 rows, 1500 keys: batch 64 207 / 217 / 367, batch 4 22.8 /
 *   21.3 / 23.3, batch 1 - / 16.0 / 11.7 (15.0 with two splits of wm 1);
 *   8 heads of 64, 1000 x 1000: 16.5 / 12.4 / 9.7 (best split 14.5);
 *   one head of 256, 5184 x 20751, bf16: 138 with 12 splits, 192 with 16 (a
 *   workgroup too many per compute unit), 175 with 8, wm 2 236, wm 8 130.
 * So: as many rows as still give two workgroups per compute unit, or one and a
 * quarter with wm 2; splits only where even the least rows leave half of the
 * compute units idle, and then two workgroups for each.
 * With up to 64 rows (tokens being made) one workgroup per compute unit is
 * enough, if that makes eight splits: one token over 8192 keys, 16 / 48 key heads
 * of 128 / 64 18.5 / 21.7, with four workgroups per compute unit 21.2 / 26.0; 12 of
 * 64 over 32768 24.3 and 31.5. Else eight, since lengths may differ: 16
 * sequences of 40 to 100 % of 8192 keys, 8 key heads of 128 78.1, four 81.0; but
 * 64 sequences of 2048 67 without and 75 with two. Down to 128 keys each: floats,
 * 10 x 700, 8 heads of 64 15.3, down to 256 21.9. */
static void plan(struct xattn_desc *d)
{
    const long cu = dev_cu_count(), rows = (long)d->grp * d->Nq;
    const int rb = padded(d->hd) * (d->dt == DT_F32 ? 4 : 2);
    /* Waves that share keys have 32 of a tile each: wider rows would leave LDS
     * for one workgroup per compute unit (step of 16 sequences above: wm 1 88
     * us, wm 2 79), or none. */
    const int least = rb >= 1024 ? 4 : rb >= 256 ? 2 : 1;
    int wm = rows > 64 ? 4 : rows > 32 ? 2 : 1;

#define WG(wm) (d->units * ((rows + 32 * (wm) - 1) / (32 * (wm))))
    if (wm < least)
        wm = least;
    d->splits = 1;
    d->few = d->vec && d->hd <= 64 && d->Nk <= 64;
    if (d->few) {
        /* Workgroups of a unit, a wave for each block of 32 rows at most. */
        long parts = 4 * cu / d->units;

        if (parts > (rows + 127) / 128)
            parts = (rows + 127) / 128;
        d->tiles = parts < 1 ? 1 : (int)parts;
        return;
    }
    if (!d->vec)
        wm = rb >= 1024 ? 4 : 2;
    if (d->vec && d->dt != DT_F32 && rb >= 256 && rows >= (rb == 256 ? 1024 : 256) && d->Nk > 256) {
        /* The copies into LDS are what such heads wait for (6 to 8 TB/s): 256 rows
         * share them, one workgroup of eight waves per compute unit and as many
         * splits as make one for each, unless they get short. us, against the
         * rules below: 5184 x 5184 with 8, 4, 2 heads of 128 127 / 71 / 45 and
         * 154 / 85 / 60; 5184 x 20751, one head of 256 130 and 138; 447 x 1500,
         * 64 heads of 256 83 and 97. But with heads of 128 2048 x 2048, 8 heads
         * in splits of 512 keys 37 and 31, 512 x 2048, 64 heads 56 and 48. */
        const long tiles = (rows + 255) / 256, wg = d->units * tiles;
        long want = cu / wg, rounds;

        if (want > d->Nk / (rb == 256 ? 768 : 384))
            want = d->Nk / (rb == 256 ? 768 : 384);
        if (want < 1)
            want = 1;
        rounds = (wg * want + cu - 1) / cu;
        /* Where more than four in ten compute units would be idle: below. */
        if (10 * wg * want >= 6 * cu * rounds) {
            d->wm = 8;
            d->tiles = (int)tiles;
            d->splits = (int)want;
            d->heads_first = 0;
            return;
        }
    }
    if (d->vec && d->dt == DT_F32 && rows > 64) {
        /* Float products fill the SIMDs, so that even loads of the compute units
         * count most: the cheapest cut. us, against the rules below: 449 x 2533,
         * 12 heads of 96 77 and 101; 1000 x 1000, 8 heads of 64 26 and 41, of
         * 128 50 and 77; 5184 x 5184, 8 heads of 128 857 and 1079. */
        static const int cuts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
        double best = 0.0;

        for (int w = 4; w >= (rb >= 1024 ? 4 : rb >= 512 ? 2 : 1); w /= 2)
            for (int n : cuts) {
                const double c = cost_f32(d, w, n, rows, cu);

                if (n > 1 && (d->Nk <= 256 || d->Nk / n < 192))
                    break;
                if (best == 0.0 || c < best) {
                    best = c;
                    wm = w;
                    d->splits = n;
                }
            }
    }
    else if (d->Nk > 256) {
        const int most_rows = wm;
        long want = 2 * cu;

        if (d->vec && wm == 4 && least <= 2 && WG(4) < 2 * cu)
            wm = 2;
        if (d->vec && wm == 2 && least == 1 && WG(2) < cu + cu / 4)
            wm = 1;
        if (rows <= 64 ? WG(wm) < 2 * cu : WG(wm) < cu / 2) {
            const int least_keys = rows <= 64 ? 128 : 384;

            wm = most_rows;
            if (rows <= 64) {
                want = cu;
                if (cu / WG(wm) < 8)
                    want = 8 * WG(wm) < 4 * cu ? 8 * WG(wm) : 4 * cu;
            }
            want /= WG(wm);
            if (want > d->Nk / least_keys)
                want = d->Nk / least_keys;
            d->splits = want < 1 ? 1 : want > 64 ? 64 : (int)want;
        }
    }
    d->wm = wm;
    d->tiles = (int)((rows + 32 * wm - 1) / (32 * wm));
    d->heads_first = d->Nk <= 256;
#undef WG
}

/* Offset of the splits' (m, sum) pairs in floats, and all of the workspace
 * in bytes. */
static size_t part_ml(const struct xattn_desc *d)
{
    return ((size_t)d->splits * d->units * d->grp * d->Nq * d->hd + 3) & ~(size_t)3;
}

static size_t part_bytes(const struct xattn_desc *d)
{
    return d->splits == 1
               ? 0
               : 4 * part_ml(d) + 8 * (size_t)d->splits * d->units * d->grp * d->Nq;
}

extern "C" size_t xattn_ws(struct xattn_desc *d)
{
    plan(d);
    return part_bytes(d);
}

template <int DT, int DP, int WM, int TK, int ST, int OCC, bool VEC = true, int DB = DP / 32>
static int run_blocks(const struct xattn_desc *d, hipStream_t s)
{
    const unsigned grid = d->heads_first ? item_grid(d->tiles, d->units)
                                         : item_grid(d->units * d->splits, d->tiles);

    hipLaunchKernelGGL((k_xattn<DT, DP, DB, WM, TK, ST, OCC, VEC>), dim3(grid),
                       dim3(WM == 8 ? 512 : 256), 0, s, *d);
    return hipGetLastError();
}

/* Heads of up to three quarters of the padded width take a kernel without the
 * last quarter's products. us, against the products of zeros: 8 heads of 96
 * bf16, 5184 x 5184 108 and 146; 2 of 192, 3000 x 3000 39 and 63; 32 of 80,
 * 1024 x 1024 24.6 and 27.0; 12 of 96 floats, 449 x 2533 97 and 126. */
template <int DT, int DP, int WM, int TK, int ST, int OCC, bool VEC = true>
static int run(const struct xattn_desc *d, hipStream_t s)
{
    if constexpr (VEC && DP >= 128)
        if (d->hd <= DP / 4 * 3)
            return run_blocks<DT, DP, WM, TK, ST, OCC, VEC, DP / 128 * 3>(d, s);
    return run_blocks<DT, DP, WM, TK, ST, OCC, VEC>(d, s);
}

template <int DT, int DP, int NB> static int run_few(const struct xattn_desc *d, hipStream_t s)
{
    hipLaunchKernelGGL((k_xattn_few<DT, DP, NB>), dim3(item_grid(d->tiles, d->units)), dim3(256), 0,
                       s, *d);
    return hipGetLastError();
}

template <int DT, int DP> static int run_wm(const struct xattn_desc *d, hipStream_t s)
{
    constexpr int RB = DP * xt<DT>::size;

    if constexpr (DP <= 64)
        if (d->few)
            return d->Nk <= 32 ? run_few<DT, DP, 1>(d, s) : run_few<DT, DP, 2>(d, s);

    if (!d->vec) {
        if constexpr (RB == 1024)
            return run<DT, DP, 4, 32, 2, 1, false>(d, s);
        else
            return run<DT, DP, 2, 64, 2, 1, false>(d, s);
    }
    if (d->wm == 8) {
        if constexpr (DT != DT_F32 && RB >= 256)
            return run<DT, DP, 8, RB == 256 ? 64 : 32, 3, 2>(d, s);
        return hipErrorInvalidValue;
    }
    /* LDS of a tile of 64 keys: 8, 16, 32 KiB for rows of 64, 128, 256 bytes. */
    if (d->wm == 4) {
        if constexpr (RB <= 128)
            return run<DT, DP, 4, 64, 3, 2>(d, s);
        else if constexpr (RB == 256)
            return run<DT, DP, 4, 64, 2, 2>(d, s);
        else if constexpr (RB == 512)
            return run<DT, DP, 4, 32, 2, 2>(d, s);
        else
            return run<DT, DP, 4, 32, 2, 1>(d, s);
    }
    if (d->wm == 2) {
        if constexpr (RB <= 256)
            return run<DT, DP, 2, 64, 2, 2>(d, s);
        else if constexpr (RB == 512)
            return run<DT, DP, 2, 64, 2, 1>(d, s);
    }
    if constexpr (RB <= 128)
        return run<DT, DP, 1, 128, 2, 2>(d, s);
    else if constexpr (RB == 256 && DT == DT_F32)
        return run<DT, DP, 1, 128, 2, 1>(d, s);
    return hipErrorInvalidValue;
}

template <int DT, int LP, bool VEC> static void merge(const struct xattn_desc *d, hipStream_t s)
{
    const long rows = (long)d->units * d->grp * d->Nq, blocks = (rows * LP + 255) / 256;

    hipLaunchKernelGGL((k_xattn_merge<DT, LP, VEC>), dim3((unsigned)blocks), dim3(256), 0, s, *d);
}

template <int DT> static int run_dt(struct xattn_desc *d, hipStream_t s)
{
    const int dp = padded(d->hd);
    int err = dp == 32    ? run_wm<DT, 32>(d, s)
              : dp == 64  ? run_wm<DT, 64>(d, s)
              : dp == 128 ? run_wm<DT, 128>(d, s)
                          : run_wm<DT, 256>(d, s);

    if (err == hipSuccess && d->splits > 1) {
        if (!d->vec)
            merge<DT, 64, false>(d, s);
        else if (dp <= 64)
            merge<DT, 16, true>(d, s);
        else
            merge<DT, 32, true>(d, s);
        err = hipGetLastError();
    }
    return err;
}

extern "C" int launch_xattn(struct xattn_desc *d, void *ws, size_t ws_bytes, void *stream)
{
    /* Without the room one workgroup per row tile walks all keys. */
    if (!ws || ws_bytes < part_bytes(d))
        d->splits = 1;
    d->part = (float *)ws;
    d->part_ml = d->splits > 1 ? (long)part_ml(d) : 0;
    if (d->dt == DT_F32)
        return run_dt<DT_F32>(d, (hipStream_t)stream);
    if (d->dt == DT_F16)
        return run_dt<DT_F16>(d, (hipStream_t)stream);
    return run_dt<DT_BF16>(d, (hipStream_t)stream);
}
