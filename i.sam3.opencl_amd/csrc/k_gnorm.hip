/* SPDX-License-Identifier: Unlicense
 *
 * Group norm of channels-last rows with affine and activation (groupnorm):
 * per (batch, group of channels) y = act((x - mean) / sqrt(var + eps) g + b),
 * mean and variance over all rows and the group's channels. Bound by HBM: the
 * input read once (its second reading comes from the caches), the output
 * written once.
 *
 * Sums of x and x^2 are kept in 64 bits: the variance is then their
 * difference without loss for means up to 10^6 deviations, millions of rows
 * and one pass.
 */
#include "k_common.h"

#define ACT_SILU_K 3

template <int DT> __device__ __forceinline__ float from(uint16_t v)
{
    return DT == DT_BF16 ? bf2f(v) : h2f(v);
}

/* V consecutive elements as floats, and back. */
template <int DT, int V> struct vec {
    float v[V];

    __device__ __forceinline__ void get(const void *base, long at)
    {
        if constexpr (DT == DT_F32) {
            const float *p = (const float *)base + at;

            if constexpr (V == 4)
                *(f32x4 *)v = *(const f32x4 *)p;
            else if constexpr (V == 2)
                *(float2 *)v = *(const float2 *)p;
            else
                v[0] = p[0];
        }
        else {
            const uint16_t *p = (const uint16_t *)base + at;
            uint16_t u[V];

            if constexpr (V == 8)
                *(u32x4 *)u = *(const u32x4 *)p;
            else if constexpr (V == 4)
                *(u32x2 *)u = *(const u32x2 *)p;
            else if constexpr (V == 2)
                *(uint32_t *)u = *(const uint32_t *)p;
            else
                u[0] = p[0];
#pragma unroll
            for (int i = 0; i < V; i++)
                v[i] = from<DT>(u[i]);
        }
    }
    __device__ __forceinline__ void put(void *base, long at) const
    {
        if constexpr (DT == DT_F32) {
            float *p = (float *)base + at;

            if constexpr (V == 4)
                *(f32x4 *)p = *(const f32x4 *)v;
            else if constexpr (V == 2)
                *(float2 *)p = *(const float2 *)v;
            else
                p[0] = v[0];
        }
        else {
            uint16_t *p = (uint16_t *)base + at;
            uint16_t u[V];

#pragma unroll
            for (int i = 0; i < V; i++)
                u[i] = DT == DT_BF16 ? f2bf(v[i]) : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
            if constexpr (V == 8)
                *(u32x4 *)p = *(const u32x4 *)u;
            else if constexpr (V == 4)
                *(u32x2 *)p = *(const u32x2 *)u;
            else if constexpr (V == 2)
                *(uint32_t *)p = *(const uint32_t *)u;
            else
                p[0] = u[0];
        }
    }
};

__device__ __forceinline__ float act_gn(float v, int act)
{
    if (act == ACT_SILU_K)
        return v / (1.0f + __expf(-v));
    /* Not fmaxf: a NaN stays one. */
    if (act == ACT_RELU_K)
        return v < 0.0f ? 0.0f : v;
    return act_k(v, act);
}

/* Mean (in two floats) and 1 / sqrt(var + eps) of n values with sum s.x and
 * sum of squares s.y. */
struct stat {
    float hi, lo, rs;
};

__device__ __forceinline__ struct stat stat_of(double2 s, double n, float eps)
{
    const double mean = s.x / n, var = s.y / n - mean * mean;
    struct stat r;

    r.hi = (float)mean;
    r.lo = (float)(mean - r.hi);
    r.rs = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps));
    return r;
}

/* One workgroup of 1024 per (group, batch): sums, then the same elements again
 * (from L2, or held in registers up to NR vectors per thread). */
template <int DT, int V>
__global__ __launch_bounds__(1024) void k_gn_group(const struct groupnorm_desc d)
{
    constexpr int NR = 32 / V;
    __shared__ double2 red[16];
    const int t = threadIdx.x, grp = blockIdx.x, b = blockIdx.y;
    const int cg = d.C / d.groups, gv = cg / V;
    const long n = d.rows * gv;
    const long xb = d.xo + b * d.xs0 + grp * cg, yb = d.yo + b * d.ys0 + grp * cg;
    double2 s = {0.0, 0.0};
    vec<DT, V> keep[NR];
    const bool held = n <= 1024L * NR;

    if (held) {
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const long i = t + 1024L * k;

            if (i < n) {
                keep[k].get(d.X, xb + i / gv * d.xld + i % gv * V);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const double x = keep[k].v[e];

                    s.x += x;
                    s.y = fma(x, x, s.y);
                }
            }
        }
    }
    else
        for (long i = t; i < n; i += 1024) {
            vec<DT, V> x;

            x.get(d.X, xb + i / gv * d.xld + i % gv * V);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const double xe = x.v[e];

                s.x += xe;
                s.y = fma(xe, xe, s.y);
            }
        }
    for (int o = 32; o > 0; o >>= 1) {
        s.x += __shfl_xor(s.x, o, 64);
        s.y += __shfl_xor(s.y, o, 64);
    }
    if ((t & 63) == 0)
        red[t >> 6] = s;
    __syncthreads();
    s = red[0];
    for (int i = 1; i < 16; i++) {
        s.x += red[i].x;
        s.y += red[i].y;
    }
    const struct stat st = stat_of(s, (double)d.rows * cg, d.eps);
    auto apply = [&](vec<DT, V> &x, long i) {
        const int c = (int)(i % gv) * V;

#pragma unroll
        for (int e = 0; e < V; e++) {
            const float g = d.g ? d.g[grp * cg + c + e] : 1.0f;
            const float be = d.b ? d.b[grp * cg + c + e] : 0.0f;

            x.v[e] = act_gn(fmaf((x.v[e] - st.hi) - st.lo, st.rs * g, be), d.act);
        }
        x.put(d.Y, yb + i / gv * d.yld + c);
    };

    if (held) {
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const long i = t + 1024L * k;

            if (i < n)
                apply(keep[k], i);
        }
    }
    else
        for (long i = t; i < n; i += 1024) {
            vec<DT, V> x;

            x.get(d.X, xb + i / gv * d.xld + i % gv * V);
            apply(x, i);
        }
}

/* Rows of chunk blockIdx.x of batch blockIdx.y. */
__device__ __forceinline__ void chunk_rows(const struct groupnorm_desc &d, long *r0, long *r1)
{
    const long per = (d.rows + d.chunks - 1) / d.chunks;

    *r0 = min(d.rows, blockIdx.x * per);
    *r1 = min(d.rows, *r0 + per);
}

/* Sums of a chunk of rows, per group. A thread keeps one column of V channels
 * (or, where a row has more than 256 of them, one of each block of 256) and
 * walks every (256 / columns)-th row; a group's threads are then added in
 * order. */
template <int DT, int V>
__global__ __launch_bounds__(256) void k_gn_stats(const struct groupnorm_desc d)
{
    __shared__ double2 red[256];
    const int t = threadIdx.x, b = blockIdx.y;
    const int cv = d.C / V, gv = d.C / d.groups / V;
    double2 *const part = (double2 *)d.part + ((long)b * d.chunks + blockIdx.x) * d.groups;
    long r0, r1;

    chunk_rows(d, &r0, &r1);
    const int w = min(cv, 256), lanes = 256 / w;
    const int col = t % w, row = t / w;

    /* Groups that reach over two blocks of columns add to what is there. */
    for (int g = t; g < d.groups; g += 256)
        part[g] = double2{0.0, 0.0};
    for (int c0 = 0; c0 < cv; c0 += w) {
        double2 s = {0.0, 0.0};
        const int c = c0 + col;

        if (c < cv && row < lanes)
#pragma unroll 4
            for (long r = r0 + row; r < r1; r += lanes) {
                vec<DT, V> x;

                x.get(d.X, d.xo + b * d.xs0 + r * d.xld + (long)c * V);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const double xe = x.v[e];

                    s.x += xe;
                    s.y = fma(xe, xe, s.y);
                }
            }
        __syncthreads();
        red[t] = s;
        __syncthreads();
        const int g0 = c0 / gv, g1 = (min(c0 + w, cv) - 1) / gv;

        for (int g = g0 + t; g <= g1; g += 256) {
            double2 q = part[g];
            const int a = max(c0, g * gv) - c0, e = min(min(c0 + w, cv), (g + 1) * gv) - c0;

            for (int k = 0; k < lanes; k++)
                for (int i = a; i < e; i++) {
                    q.x += red[k * w + i].x;
                    q.y += red[k * w + i].y;
                }
            part[g] = q;
        }
    }
}

/* The chunk's rows normalised: mean and deviation of each group from the
 * sums of all chunks, in order. */
template <int DT, int V>
__global__ __launch_bounds__(256) void k_gn_apply(const struct groupnorm_desc d)
{
    extern __shared__ struct stat st[];
    const int t = threadIdx.x, b = blockIdx.y;
    const int cg = d.C / d.groups, cv = d.C / V, gv = cg / V;
    const double2 *const part = (const double2 *)d.part + (long)b * d.chunks * d.groups;
    long r0, r1;

    chunk_rows(d, &r0, &r1);
    for (int g = t >> 6; g < d.groups; g += 4) {
        double2 s = {0.0, 0.0};

        for (int k = t & 63; k < d.chunks; k += 64) {
            const double2 x = part[(long)k * d.groups + g];

            s.x += x.x;
            s.y += x.y;
        }
        for (int o = 32; o > 0; o >>= 1) {
            s.x += __shfl_xor(s.x, o, 64);
            s.y += __shfl_xor(s.y, o, 64);
        }
        if ((t & 63) == 0)
            st[g] = stat_of(s, (double)d.rows * cg, d.eps);
    }
    __syncthreads();
    const int w = min(cv, 256), lanes = 256 / w;
    const int col = t % w, row = t / w;

    for (int c = col; c < cv && row < lanes; c += w) {
        const struct stat q = st[c / gv];
        float a[V], be[V];

#pragma unroll
        for (int e = 0; e < V; e++) {
            a[e] = q.rs * (d.g ? d.g[c * V + e] : 1.0f);
            be[e] = d.b ? d.b[c * V + e] : 0.0f;
        }
#pragma unroll 4
        for (long r = r0 + row; r < r1; r += lanes) {
            vec<DT, V> x;

            x.get(d.X, d.xo + b * d.xs0 + r * d.xld + (long)c * V);
#pragma unroll
            for (int e = 0; e < V; e++)
                x.v[e] = act_gn(fmaf((x.v[e] - q.hi) - q.lo, a[e], be[e]), d.act);
            x.put(d.Y, d.yo + b * d.ys0 + r * d.yld + (long)c * V);
        }
    }
}

/* ------------------------------------------------------------ launch */

/* Row chunks per batch entry, or 1: one workgroup per group then holds its
 * elements (32 per thread) or the whole is small. */
static void plan(struct groupnorm_desc *d)
{
    const long elems = d->rows * (d->C / d->groups);
    const int cu = dev_cu_count();
    long chunks = 1;

    if (elems > 32 * 1024) {
        chunks = (4L * cu + d->nb - 1) / d->nb;
        if (chunks > d->rows / 8)
            chunks = d->rows / 8;
        if (chunks > 1024)
            chunks = 1024;
        if (chunks < 1)
            chunks = 1;
    }
    d->chunks = (int)chunks;
}

extern "C" size_t groupnorm_ws_bytes(struct groupnorm_desc *d)
{
    plan(d);
    return d->chunks > 1 ? 16 * (size_t)d->nb * d->chunks * d->groups : 0;
}

template <int DT, int V> static int run(const struct groupnorm_desc *d, hipStream_t s)
{
    if (d->chunks == 1)
        hipLaunchKernelGGL((k_gn_group<DT, V>), dim3(d->groups, d->nb), dim3(1024), 0, s, *d);
    else {
        hipLaunchKernelGGL((k_gn_stats<DT, V>), dim3(d->chunks, d->nb), dim3(256), 0, s, *d);
        if (hipGetLastError() != hipSuccess)
            return hipErrorLaunchFailure;
        hipLaunchKernelGGL((k_gn_apply<DT, V>), dim3(d->chunks, d->nb), dim3(256),
                           d->groups * sizeof(struct stat), s, *d);
    }
    return hipGetLastError();
}

template <int DT> static int run_dt(const struct groupnorm_desc *d, hipStream_t s)
{
    if constexpr (DT != DT_F32)
        if (d->vec == 8)
            return run<DT, 8>(d, s);
    if (d->vec >= 4)
        return run<DT, 4>(d, s);
    return d->vec == 2 ? run<DT, 2>(d, s) : run<DT, 1>(d, s);
}

extern "C" int launch_groupnorm(struct groupnorm_desc *d, void *ws, size_t ws_bytes, void *stream)
{
    const size_t need = groupnorm_ws_bytes(d);

    if (need && (!ws || ws_bytes < need))
        d->chunks = 1;
    d->part = (float *)ws;
    return d->dt == DT_F32   ? run_dt<DT_F32>(d, (hipStream_t)stream)
           : d->dt == DT_F16 ? run_dt<DT_F16>(d, (hipStream_t)stream)
                             : run_dt<DT_BF16>(d, (hipStream_t)stream);
}
