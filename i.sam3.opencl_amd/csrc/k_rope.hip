/* SPDX-License-Identifier: Unlicense
 *
 * Rotary positions: the (cos, sin) tables that the attention reads
 * (rope_table) and the rotation of rows by them (rope_rows). Both are bound
 * by HBM: a table is written once, a row read and written once.
 */
#include "k_common.h"

/* Workgroups per compute unit beyond which a thread takes more rows (tables) or
 * heads, and heads whose loads are under way together. us with 2 / 4 / 8 heads:
 * 32774 rows of 8 x 128 halves 36.4 / 33.8 / 32.3; a table of 131072 x 64 pairs
 * the same within 3 % from 8 to 32 workgroups. */
#define TABLE_WG 16
#define ROWS_WG 8L
#define HEADS_AHEAD 4

/* Results go past the caches: written through them, the lines are held until
 * the kernel's end and go out then. The rows above take 23.2 us (139 MB, 6.0
 * TB/s) for 33.8, the table 13.3 (67 MB) for 14.2. */
#define STORE(p, x) __builtin_nontemporal_store(x, p)

/* ------------------------------------------------------------ tables */

/* cos and sin of a turn's fraction. Whole turns and quarters come off in 64
 * bits (exactly: the products that follow are by 4 and 1/4), the rest, at most
 * an eighth of a turn, goes through the Taylor series in 32 bits, whose
 * next terms are below 2e-9 (sin) and 2e-10 (cos) at pi / 4. */
__device__ __forceinline__ float2 cos_sin_turns(double t)
{
    const double r = t - __builtin_rint(t);
    const double k = __builtin_rint(4.0 * r);
    const float x = 6.28318530717958648f * (float)(r - 0.25 * k), x2 = x * x;
    const int q = (int)k;
    float s = 1.0f / 362880, c = -1.0f / 3628800;

    s = fmaf(s, x2, -1.0f / 5040);
    s = fmaf(s, x2, 1.0f / 120);
    s = fmaf(s, x2, -1.0f / 6);
    s = fmaf(s * x2, x, x);
    c = fmaf(c, x2, 1.0f / 40320);
    c = fmaf(c, x2, -1.0f / 720);
    c = fmaf(c, x2, 1.0f / 24);
    c = fmaf(c, x2, -0.5f);
    c = fmaf(c, x2, 1.0f);
    const float a = q & 1 ? s : c, b = q & 1 ? c : s;

    /* Quarters q = -2 .. 2: cos changes sign for 1, 2, -2, sin for 2, -1, -2. */
    return float2{(q + 1) & 2 ? -a : a, q & 2 ? -b : b};
}

/* A thread keeps one pair (or two where their number is even, so that it
 * writes 16 bytes) and walks rows blockIdx.y step apart. */
template <int N> __global__ __launch_bounds__(256) void k_rope_table(const struct rope_table_desc d)
{
    const int units = d.pairs / N, per = 256 / min(units, 256);
    const int t = threadIdx.x, u = blockIdx.x * 256 + t % min(units, 256);

    if (u >= units || t / min(units, 256) >= per)
        return;
    double f[N];

#pragma unroll
    for (int e = 0; e < N; e++)
        f[e] = d.turns[u * N + e];
    for (long p = blockIdx.y * per + t / min(units, 256); p < d.npos; p += gridDim.y * per) {
        const int pos = d.pos ? d.pos[p] : (int)p;
        float v[2 * N];

#pragma unroll
        for (int e = 0; e < N; e++) {
            const int at = !d.W ? pos : u * N + e < d.pairs / 2 ? pos % d.W : pos / d.W;
            const float2 cs = cos_sin_turns(at * f[e]);

            v[2 * e] = cs.x * d.mul;
            v[2 * e + 1] = cs.y * d.mul;
        }
        float *const o = d.table + 2 * (p * d.pairs + u * N);

        if constexpr (N == 2)
            STORE((f32x4 *)o, (f32x4{v[0], v[1], v[2], v[3]}));
        else
            *(float2 *)o = float2{v[0], v[1]};
    }
}

extern "C" int launch_rope_table(const struct rope_table_desc *d, void *stream)
{
    const int n = d->pairs % 2 == 0 && (uintptr_t)d->table % 16 == 0 ? 2 : 1;
    const int units = d->pairs / n, per = 256 / (units < 256 ? units : 256);
    long y = ((long)d->npos + per - 1) / per;

    if (y > TABLE_WG * dev_cu_count())
        y = TABLE_WG * dev_cu_count();
    const dim3 grid((unsigned)((units + 255) / 256), (unsigned)y);

    if (n == 2)
        hipLaunchKernelGGL(k_rope_table<2>, grid, dim3(256), 0, (hipStream_t)stream, *d);
    else
        hipLaunchKernelGGL(k_rope_table<1>, grid, dim3(256), 0, (hipStream_t)stream, *d);
    return hipGetLastError();
}

/* ------------------------------------------------------------ rows */

template <int DT> __device__ __forceinline__ float from(uint16_t v)
{
    return DT == DT_BF16 ? bf2f(v) : h2f(v);
}

template <int DT> __device__ __forceinline__ uint16_t to(float v)
{
    return DT == DT_BF16 ? f2bf(v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

/* N elements at p as floats, and back. */
template <int DT, int N> __device__ __forceinline__ void get(const char *p, float *v)
{
    if constexpr (DT == DT_F32) {
        if constexpr (N == 4)
            *(f32x4 *)v = *(const f32x4 *)p;
        else
            for (int i = 0; i < N; i++)
                v[i] = ((const float *)p)[i];
    }
    else {
        uint16_t u[N];

        if constexpr (N == 8)
            *(u32x4 *)u = *(const u32x4 *)p;
        else
            for (int i = 0; i < N; i++)
                u[i] = ((const uint16_t *)p)[i];
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] = from<DT>(u[i]);
    }
}

template <int DT, int N> __device__ __forceinline__ void put(char *p, const float *v)
{
    if constexpr (DT == DT_F32) {
        if constexpr (N == 4)
            STORE((f32x4 *)p, *(const f32x4 *)v);
        else
            for (int i = 0; i < N; i++)
                ((float *)p)[i] = v[i];
    }
    else {
        uint16_t u[N];

#pragma unroll
        for (int i = 0; i < N; i++)
            u[i] = to<DT>(v[i]);
        if constexpr (N == 8)
            STORE((u32x4 *)p, *(const u32x4 *)u);
        else
            for (int i = 0; i < N; i++)
                ((uint16_t *)p)[i] = u[i];
    }
}

/* A thread per (row, unit), over the heads blockIdx.y, blockIdx.y +
 * gridDim.y, ...: the table's values are read once for all of them. A unit is
 * N columns: HALVES takes N columns of the first half of the rotated part and
 * their partners, !HALVES N / 2 pairs (one where N is 1); the units behind
 * are copied. */
template <int DT, int N, bool HALVES>
__global__ __launch_bounds__(256) void k_rope_rows(const struct rope_rows_desc d, int units,
                                                   int turned)
{
    constexpr int S = DT == DT_F32 ? 4 : 2;
    constexpr int M = HALVES ? N : N == 1 ? 2 : N; /* columns of a unit at one place */
    constexpr int P = HALVES ? N : M / 2;          /* pairs of a unit */
    const long i = (long)blockIdx.x * 256 + threadIdx.x;

    if (i >= (long)d.nb * d.rows * units)
        return;
    const int u = (int)(i % units);
    const long row = i / units;
    const int b = (int)(row / d.rows), r = (int)(row % d.rows);
    const long p = d.pos ? (long)d.pos[row] : (d.pos0 + r) % d.npos;
    const bool turn = u < turned && p >= 0 && p < d.npos;
    const char *x = (const char *)d.X + S * (d.xo + b * d.xs0 + (long)r * d.xld);
    char *y = (char *)d.Y + S * (d.yo + b * d.ys0 + (long)r * d.yld);

    if (u >= turned) {
        /* Columns behind the rotated ones. */
        if (!d.copy)
            return;
        const int c = d.rot + (u - turned) * N;

        for (int h = blockIdx.y; h < d.heads; h += gridDim.y) {
            float v[N];

            get<DT, N>(x + S * (h * d.xs1 + c), v);
            put<DT, N>(y + S * (h * d.ys1 + c), v);
        }
        return;
    }
    const int c0 = HALVES ? u * N : u * M, c1 = c0 + d.rot / 2;
    float cs[2 * P];

    if (turn) {
        const float *t = d.table + 2 * (p * (d.rot / 2) + u * P);

#pragma unroll
        for (int k = 0; k < P; k++)
            *(float2 *)(cs + 2 * k) = ((const float2 *)t)[k];
    }
    else {
#pragma unroll
        for (int k = 0; k < P; k++) {
            cs[2 * k] = 1.0f;
            cs[2 * k + 1] = 0.0f;
        }
        if (!d.copy)
            return;
    }
    for (int h0 = blockIdx.y; h0 < d.heads; h0 += HEADS_AHEAD * gridDim.y) {
        float v[HEADS_AHEAD][2 * P];

#pragma unroll
        for (int j = 0; j < HEADS_AHEAD; j++) {
            const char *xh = x + S * (min(h0 + j * (int)gridDim.y, d.heads - 1) * d.xs1);

            if (HALVES) {
                get<DT, N>(xh + S * c0, v[j]);
                get<DT, N>(xh + S * c1, v[j] + N);
            }
            else
                get<DT, M>(xh + S * c0, v[j]);
        }
#pragma unroll
        for (int j = 0; j < HEADS_AHEAD; j++) {
            const int h = h0 + j * gridDim.y;
            char *yh = y + S * (h * d.ys1);
            float o[2 * P];

            if (h >= d.heads)
                break;
#pragma unroll
            for (int k = 0; k < P; k++) {
                const int ia = HALVES ? k : 2 * k, ib = HALVES ? N + k : 2 * k + 1;
                const float c = cs[2 * k], s = cs[2 * k + 1];

                o[ia] = turn ? fmaf(v[j][ia], c, -(v[j][ib] * s)) : v[j][ia];
                o[ib] = turn ? fmaf(v[j][ia], s, v[j][ib] * c) : v[j][ib];
            }
            if (HALVES) {
                put<DT, N>(yh + S * c0, o);
                put<DT, N>(yh + S * c1, o + N);
            }
            else
                put<DT, M>(yh + S * c0, o);
        }
    }
}

template <int DT, int N, bool HALVES>
static int run(const struct rope_rows_desc *d, hipStream_t s)
{
    const int turned = HALVES ? d->rot / 2 / N : d->rot / (N == 1 ? 2 : N);
    const int units = turned + (d->hd - d->rot) / N;
    const long n = (long)d->nb * d->rows * units;
    const long blocks = (n + 255) / 256;
    /* Heads are spread over workgroups until the device is full. */
    long hy = (ROWS_WG * dev_cu_count() + blocks - 1) / blocks;

    if (hy > d->heads)
        hy = d->heads;
    hipLaunchKernelGGL((k_rope_rows<DT, N, HALVES>), dim3((unsigned)blocks, (unsigned)hy),
                       dim3(256), 0, s, *d, units, turned);
    return hipGetLastError();
}

template <int DT> static int run_dt(const struct rope_rows_desc *d, hipStream_t s)
{
    constexpr int V = DT == DT_F32 ? 4 : 8;

    if (d->halves)
        return d->vec ? run<DT, V, true>(d, s) : run<DT, 1, true>(d, s);
    return d->vec ? run<DT, V, false>(d, s) : run<DT, 1, false>(d, s);
}

extern "C" int launch_rope_rows(const struct rope_rows_desc *d, void *stream)
{
    hipStream_t s = (hipStream_t)stream;

    return d->dt == DT_F32   ? run_dt<DT_F32>(d, s)
           : d->dt == DT_F16 ? run_dt<DT_F16>(d, s)
                             : run_dt<DT_BF16>(d, s);
}
