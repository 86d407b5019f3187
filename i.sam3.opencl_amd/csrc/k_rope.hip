/* SPDX-License-Identifier: Unlicense
 *
 * Rotary positions: the (cos, sin) tables that the attention reads
 * (rope_table) and the rotation of rows by them (rope_rows). Both are bound
 * by HBM: a table is written once, a row read and written once.
 */
#include "k_common.h"

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

/* A thread per angle, pairs fastest: consecutive lanes write consecutive
 * (cos, sin). */
__global__ __launch_bounds__(256) void k_rope_table(const struct rope_table_desc d)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;

    if (i >= (long)d.npos * d.pairs)
        return;
    const int p = (int)(i / d.pairs), j = (int)(i % d.pairs);
    int pos = d.pos ? d.pos[p] : p;

    if (d.W)
        pos = j < d.pairs / 2 ? pos % d.W : pos / d.W;
    const float2 cs = cos_sin_turns(pos * d.turns[j]);

    ((float2 *)d.table)[i] = float2{cs.x * d.mul, cs.y * d.mul};
}

extern "C" int launch_rope_table(const struct rope_table_desc *d, void *stream)
{
    const long n = (long)d->npos * d->pairs;

    hipLaunchKernelGGL(k_rope_table, dim3((unsigned)((n + 255) / 256)), dim3(256), 0,
                       (hipStream_t)stream, *d);
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
            *(f32x4 *)p = *(const f32x4 *)v;
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
            *(u32x4 *)p = *(const u32x4 *)u;
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
#pragma unroll 4
    for (int h = blockIdx.y; h < d.heads; h += gridDim.y) {
        float v[2 * P], o[2 * P];
        const char *xh = x + S * (h * d.xs1);
        char *yh = y + S * (h * d.ys1);

        if (HALVES) {
            get<DT, N>(xh + S * c0, v);
            get<DT, N>(xh + S * c1, v + N);
        }
        else
            get<DT, M>(xh + S * c0, v);
#pragma unroll
        for (int k = 0; k < P; k++) {
            const int ia = HALVES ? k : 2 * k, ib = HALVES ? N + k : 2 * k + 1;
            const float c = cs[2 * k], s = cs[2 * k + 1];

            o[ia] = turn ? fmaf(v[ia], c, -(v[ib] * s)) : v[ia];
            o[ib] = turn ? fmaf(v[ia], s, v[ib] * c) : v[ib];
        }
        if (HALVES) {
            put<DT, N>(yh + S * c0, o);
            put<DT, N>(yh + S * c1, o + N);
        }
        else
            put<DT, M>(yh + S * c0, o);
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
    long hy = (8L * dev_cu_count() + blocks - 1) / blocks;

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
