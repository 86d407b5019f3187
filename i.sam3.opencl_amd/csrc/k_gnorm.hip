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
/* Threads of the kernels that share a batch entry's rows, and vectors that each
 * has under way. us of both kernels at 82944 rows of 256 floats, the second
 * from the first rows on: 512 threads, two workgroups per compute unit for the
 * sums, one for the rest 17.4 + 28.3; 256 threads and four 15.8 + 37; 1024 and
 * one 20.0 + 28.5 (every workgroup of the second kernel adds up all sums of
 * its batch entry). */
#define TH 512
#define AHEAD_SUMS 4
#define AHEAD_APPLY 8
/* Elements of a group that one workgroup takes, where a row's part of the
 * group is at least 16 bytes, and below that, where it reads lines for few
 * bytes of them. us by one workgroup per group and split: 8 groups of 32
 * halves, 400 rows 7.0 and 12.3, 1000 rows 13.0 and 13.2; 32 groups of 10
 * floats, 1200 rows 8.9 and 14.6; 256 groups of one float, 5000 rows 59 and
 * 23. */
#define SPLIT_ABOVE (16 * 1024)
#define SPLIT_ABOVE_NARROW (4 * 1024)

template <int DT> __device__ __forceinline__ float from(uint16_t v)
{
    return DT == DT_BF16 ? bf2f(v) : h2f(v);
}

template <int BYTES> struct raw_of;
template <> struct raw_of<16> {
    typedef u32x4 type;
};
template <> struct raw_of<8> {
    typedef u32x2 type;
};
template <> struct raw_of<4> {
    typedef uint32_t type;
};
template <> struct raw_of<2> {
    typedef uint16_t type;
};

/* V consecutive elements as they are stored, and as floats. */
template <int DT, int V> struct vec {
    static constexpr int size = DT == DT_F32 ? 4 : 2;
    typedef typename raw_of<V * size>::type raw;
    float v[V];

    __device__ __forceinline__ void set(raw r)
    {
        if constexpr (DT == DT_F32)
            __builtin_memcpy(v, &r, sizeof r);
        else {
            uint16_t u[V];

            __builtin_memcpy(u, &r, sizeof r);
#pragma unroll
            for (int i = 0; i < V; i++)
                v[i] = from<DT>(u[i]);
        }
    }
    __device__ __forceinline__ void get(const void *base, long at)
    {
        set(*(const raw *)((const char *)base + size * at));
    }
    /* Past the caches: the next kernel's reads of the input would otherwise
     * wait for these lines to be written back. */
    __device__ __forceinline__ void put(void *base, long at) const
    {
        raw r;

        if constexpr (DT == DT_F32)
            __builtin_memcpy(&r, v, sizeof r);
        else {
            uint16_t u[V];

#pragma unroll
            for (int i = 0; i < V; i++)
                u[i] = DT == DT_BF16 ? f2bf(v[i]) : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
            __builtin_memcpy(&r, u, sizeof r);
        }
        __builtin_nontemporal_store(r, (raw *)((char *)base + size * at));
    }
};

template <int ACT> __device__ __forceinline__ float act_gn(float v)
{
    if (ACT == ACT_SILU_K)
        return v / (1.0f + __expf(-v));
    /* Not fmaxf: a NaN stays one. */
    if (ACT == ACT_RELU_K)
        return v < 0.0f ? 0.0f : v;
    return act_k(v, ACT);
}

template <int A> struct act_of {
    static constexpr int value = A;
};

/* f called with the activation as a type, outside its loops. */
template <typename F> __device__ __forceinline__ void with_act(int act, F f)
{
    if (act == ACT_RELU_K)
        f(act_of<ACT_RELU_K>{});
    else if (act == ACT_GELU_K)
        f(act_of<ACT_GELU_K>{});
    else if (act == ACT_SILU_K)
        f(act_of<ACT_SILU_K>{});
    else
        f(act_of<ACT_NONE_K>{});
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

/* Vector t, t + T, ... of a group's rows, gv vectors each. */
template <int T> struct walk {
    long row;
    int col, drow, dcol, gv;

    __device__ __forceinline__ walk(unsigned t, unsigned vectors) : gv(vectors)
    {
        row = t / vectors;
        col = t % vectors;
        drow = T / vectors;
        dcol = T % vectors;
    }
    __device__ __forceinline__ void next()
    {
        row += drow;
        col += dcol;
        if (col >= gv) {
            col -= gv;
            row++;
        }
    }
};

/* One workgroup of T per (group, batch): sums, then the same elements again:
 * up to NR vectors per thread, held in registers with their g and b (which are
 * read while the sums are added up), or from the caches (NR = 0). */
template <int DT, int V, int T, int NR>
__global__ __launch_bounds__(T) void k_gn_group(const struct groupnorm_desc d)
{
    __shared__ double2 red[T / 64];
    const int t = threadIdx.x, grp = blockIdx.x, b = blockIdx.y;
    const int cg = d.C / d.groups, gv = cg / V;
    const long xb = d.xo + b * d.xs0 + (long)grp * cg, yb = d.yo + b * d.ys0 + (long)grp * cg;
    double2 s = {0.0, 0.0};
    vec<DT, V> keep[NR + 1];
    float ga[NR + 1][V], be[NR + 1][V];
    auto add = [&](const vec<DT, V> &x) {
#pragma unroll
        for (int e = 0; e < V; e++) {
            const double xe = x.v[e];

            s.x += xe;
            s.y = fma(xe, xe, s.y);
        }
    };
    auto affine = [&](int col, float *g, float *be) {
#pragma unroll
        for (int e = 0; e < V; e++) {
            g[e] = d.g ? d.g[grp * cg + col * V + e] : 1.0f;
            be[e] = d.b ? d.b[grp * cg + col * V + e] : 0.0f;
        }
    };
    walk<T> at(t, gv);

    if constexpr (NR > 0) {
#pragma unroll
        for (int k = 0; k < NR; k++, at.next())
            if (at.row < d.rows)
                keep[k].get(d.X, xb + at.row * d.xld + at.col * V);
        at = walk<T>(t, gv);
#pragma unroll
        for (int k = 0; k < NR; k++, at.next())
            if (at.row < d.rows)
                affine(at.col, ga[k], be[k]);
        at = walk<T>(t, gv);
#pragma unroll
        for (int k = 0; k < NR; k++, at.next())
            if (at.row < d.rows)
                add(keep[k]);
    }
    else
        for (; at.row < d.rows; at.next()) {
            vec<DT, V> x;

            x.get(d.X, xb + at.row * d.xld + at.col * V);
            add(x);
        }
    for (int o = 32; o > 0; o >>= 1) {
        s.x += __shfl_xor(s.x, o, 64);
        s.y += __shfl_xor(s.y, o, 64);
    }
    if ((t & 63) == 0)
        red[t >> 6] = s;
    __syncthreads();
    s = red[0];
    for (int i = 1; i < T / 64; i++) {
        s.x += red[i].x;
        s.y += red[i].y;
    }
    const struct stat st = stat_of(s, (double)d.rows * cg, d.eps);

    with_act(d.act, [&](auto act) {
        auto apply = [&](vec<DT, V> &x, const float *g, const float *be) {
#pragma unroll
            for (int e = 0; e < V; e++)
                x.v[e] = act_gn<decltype(act)::value>(
                    fmaf((x.v[e] - st.hi) - st.lo, st.rs * g[e], be[e]));
            x.put(d.Y, yb + at.row * d.yld + at.col * V);
        };

        at = walk<T>(t, gv);
        if constexpr (NR > 0) {
#pragma unroll
            for (int k = 0; k < NR; k++, at.next())
                if (at.row < d.rows)
                    apply(keep[k], ga[k], be[k]);
        }
        else
            for (; at.row < d.rows; at.next()) {
                vec<DT, V> x;

                x.get(d.X, xb + at.row * d.xld + at.col * V);
                affine(at.col, ga[0], be[0]);
                apply(x, ga[0], be[0]);
            }
    });
}

/* Chunk i of n of a batch entry's rows. */
__device__ __forceinline__ void chunk_rows(const struct groupnorm_desc &d, int n, int i, long *r0,
                                           long *r1)
{
    const long per = (d.rows + n - 1) / n;

    *r0 = min(d.rows, i * per);
    *r1 = min(d.rows, *r0 + per);
}

/* n vectors, `step` elements apart from element `at` of p, of which the next
 * AHEAD are under way. */
template <int DT, int V, int AHEAD> struct stream {
    typedef typename vec<DT, V>::raw raw;
    const char *p;
    long step, n;
    raw x[AHEAD];

    __device__ __forceinline__ raw load(long k) const
    {
        return *(const raw *)(p + min(k, n - 1) * step);
    }
    __device__ __forceinline__ void start(const void *base, long at, long step_, long n_)
    {
        p = (const char *)base + vec<DT, V>::size * at;
        step = vec<DT, V>::size * step_;
        n = n_;
        if (n > 0)
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                x[i] = load(i);
    }
    /* f on each, with its number. */
    template <typename F> __device__ __forceinline__ void run(F f)
    {
        for (long k = 0; k < n; k += AHEAD)
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                if (k + i < n) {
                    vec<DT, V> v;

                    v.set(x[i]);
                    if (k + i + AHEAD < n)
                        x[i] = load(k + i + AHEAD);
                    f(v, k + i);
                }
    }
};

/* Sums of a chunk of rows, per group. A thread keeps one column of V channels
 * (or, where a row has more than TH of them, one of each block of TH) and
 * walks every (TH / columns)-th row; a group's threads are then added in
 * order. Where the number of chunks is a multiple of 16, chunks 2 i and 2 i + 1
 * are summed on the XCD (workgroup index mod 8) whose workgroup i of k_gn_apply
 * takes both. */
template <int DT, int V>
__global__ __launch_bounds__(TH) void k_gn_stats(const struct groupnorm_desc d)
{
    __shared__ double2 red[TH];
    const int t = threadIdx.x, b = blockIdx.y;
    const int cv = d.C / V, gv = d.C / d.groups / V;
    const int i = blockIdx.x;
    const int chunk = d.chunks % 16 ? i : (i & ~15) + 2 * (i & 7) + (i >> 3 & 1);
    double2 *const part = (double2 *)d.part + (long)b * d.groups * d.chunks + chunk;
    long r0, r1;

    chunk_rows(d, d.chunks, chunk, &r0, &r1);
    const int w = min(cv, TH), lanes = TH / w;
    const int col = t % w, row = t / w;

    for (int c0 = 0; c0 < cv; c0 += w) {
        double2 s = {0.0, 0.0};
        const int c = c0 + col;

        if (c < cv && row < lanes) {
            stream<DT, V, AHEAD_SUMS> in;

            in.start(d.X, d.xo + b * d.xs0 + (r0 + row) * d.xld + (long)c * V,
                     (long)lanes * d.xld, (r1 - r0 - row + lanes - 1) / lanes);
            in.run([&](vec<DT, V> &x, long) {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const double xe = x.v[e];

                    s.x += xe;
                    s.y = fma(xe, xe, s.y);
                }
            });
        }
        __syncthreads();
        red[t] = s;
        __syncthreads();
        /* The threads of a group (columns a to e of every row), by 16 lanes. */
        const int g0 = c0 / gv, g1 = (min(c0 + w, cv) - 1) / gv;

        for (int g = g0 + t / 16; g <= g1; g += TH / 16) {
            const int a = max(c0, g * gv) - c0, e = min(min(c0 + w, cv), (g + 1) * gv) - c0;
            double2 q = {0.0, 0.0};

            for (int j = t % 16, k = j / (e - a), i = j % (e - a); k < lanes;) {
                q.x += red[k * w + a + i].x;
                q.y += red[k * w + a + i].y;
                i += 16;
                while (i >= e - a) {
                    i -= e - a;
                    k++;
                }
            }
            for (int o = 8; o > 0; o >>= 1) {
                q.x += __shfl_xor(q.x, o, 16);
                q.y += __shfl_xor(q.y, o, 16);
            }
            if (t % 16 == 0) {
                /* Groups that reach over two blocks of columns add to what is
                 * there. */
                if (c0 > g * gv) {
                    q.x += part[(long)g * d.chunks].x;
                    q.y += part[(long)g * d.chunks].y;
                }
                part[(long)g * d.chunks] = q;
            }
        }
    }
}

/* A group's sums over all chunks, in order, by a wave. */
__device__ __forceinline__ struct stat group_stat(const struct groupnorm_desc &d, int b, int g)
{
    const double2 *const p = (const double2 *)d.part + ((long)b * d.groups + g) * d.chunks;
    double2 s = {0.0, 0.0};

    for (int k = threadIdx.x & 63; k < d.chunks; k += 64) {
        const double2 x = p[k];

        s.x += x.x;
        s.y += x.y;
    }
    for (int o = 32; o > 0; o >>= 1) {
        s.x += __shfl_xor(s.x, o, 64);
        s.y += __shfl_xor(s.y, o, 64);
    }
    return stat_of(s, (double)d.rows * (d.C / d.groups), d.eps);
}

/* Where there are many sums, they are added up once. */
__global__ __launch_bounds__(256) void k_gn_sums(const struct groupnorm_desc d)
{
    const int g = blockIdx.x * 4 + (threadIdx.x >> 6), b = blockIdx.y;

    if (g >= d.groups)
        return;
    const struct stat s = group_stat(d, b, g);

    if ((threadIdx.x & 63) == 0)
        ((struct stat *)d.stats)[b * d.groups + g] = s;
}

/* The rows of two chunks normalised by mean and deviation of each group, from
 * their last ones back, half of the threads on each chunk: the rows that
 * k_gn_stats read last are still in this XCD's L2. us of both kernels at 82944
 * rows of 256 floats and 4 x 20736 of 256 bf16: 42.3 and 27.0; from the first
 * rows on 44.8 and 28.7. */
template <int DT, int V>
__global__ __launch_bounds__(TH) void k_gn_apply(const struct groupnorm_desc d)
{
    extern __shared__ struct stat st[];
    const int t = threadIdx.x, b = blockIdx.y;
    const int cv = d.C / V, gv = d.C / d.groups / V;
    long r0, r1;

    const int w = min(cv, TH), all = TH / w;
    const int two = all % 2 == 0, lanes = two ? all / 2 : all;
    const int col = t % w, row = two ? t / w >> 1 : t / w;

    if (two)
        chunk_rows(d, d.chunks, 2 * blockIdx.x + (t / w & 1), &r0, &r1);
    else
        chunk_rows(d, d.chunks / 2, blockIdx.x, &r0, &r1);
    const long n = row < lanes ? (r1 - r0 - row + lanes - 1) / lanes : 0;
    const long last = r0 + row + (n - 1) * lanes;
    stream<DT, V, AHEAD_APPLY> in;

    /* The first rows, on their way during the sums. */
    in.start(d.X, d.xo + b * d.xs0 + last * d.xld + (long)col * V, -(long)lanes * d.xld, n);
    if (d.stats)
        for (int g = t; g < d.groups; g += TH)
            st[g] = ((const struct stat *)d.stats)[b * d.groups + g];
    else
        for (int g = t >> 6; g < d.groups; g += TH / 64) {
            const struct stat q = group_stat(d, b, g);

            if ((t & 63) == 0)
                st[g] = q;
        }
    __syncthreads();
    for (int c = col; c < cv && n > 0; c += w) {
        if (c != col)
            in.start(d.X, d.xo + b * d.xs0 + last * d.xld + (long)c * V, -(long)lanes * d.xld, n);
        const struct stat q = st[c / gv];
        float a[V], be[V];

#pragma unroll
        for (int e = 0; e < V; e++) {
            a[e] = q.rs * (d.g ? d.g[c * V + e] : 1.0f);
            be[e] = d.b ? d.b[c * V + e] : 0.0f;
        }
        with_act(d.act, [&](auto act) {
            char *y = (char *)d.Y +
                      vec<DT, V>::size * (d.yo + b * d.ys0 + last * d.yld + (long)c * V);
            const long ystep = -(long)lanes * d.yld;

            in.run([&](vec<DT, V> &x, long k) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    x.v[e] = act_gn<decltype(act)::value>(
                        fmaf((x.v[e] - q.hi) - q.lo, a[e], be[e]));
                x.put(y, k * ystep);
            });
        });
    }
}

/* ------------------------------------------------------------ launch */

/* Row chunks per batch entry, or 1: one workgroup per group. */
static void plan(struct groupnorm_desc *d)
{
    const long elems = d->rows * (d->C / d->groups);
    const int cu = dev_cu_count();
    long chunks = 1;

    if (elems > (d->C / d->groups * (d->dt == DT_F32 ? 4 : 2) < 16 ? SPLIT_ABOVE_NARROW : SPLIT_ABOVE)) {
        /* Two workgroups per compute unit, none left over: 3, 7, 40 batches of
         * 20736 rows of 256 bf16 22.5, 38.5, 250 us; with those that ceil(512 /
         * batches) has 34, 59, 317. Beyond as many batches as compute units
         * several rounds even out: 300 of 5184 rows 493, with two chunks 564. */
        chunks = 2L * cu / d->nb;
        if (chunks < 2)
            chunks = 16L * cu / d->nb;
        /* Two vectors of eight per thread. */
        if (chunks > d->rows * d->C / (16 * TH))
            chunks = d->rows * d->C / (16 * TH);
        if (chunks > d->rows)
            chunks = d->rows;
        /* Pairs; and XCDs that match (see k_gn_stats) where that idles at most
         * a fifth: 17 batches 84.7 and, in 16 chunks for 30, 100.7; 7 batches
         * 42.3 in 72 chunks, 38.5 in 64. */
        chunks &= chunks >= 64 ? ~15L : ~1L;
        if (chunks < 2)
            chunks = 2;
    }
    d->chunks = (int)chunks;
}

static size_t part_bytes(const struct groupnorm_desc *d)
{
    return d->chunks > 1
               ? (size_t)d->nb * d->groups * (16 * (size_t)d->chunks + sizeof(struct stat))
               : 0;
}

extern "C" size_t groupnorm_ws_bytes(struct groupnorm_desc *d)
{
    plan(d);
    return part_bytes(d);
}

template <int DT, int V> static int run(const struct groupnorm_desc *d, hipStream_t s)
{
    const dim3 grid(d->groups, d->nb);
    int err;

    if (d->chunks == 1) {
        if (d->rows * (d->C / d->groups) <= 256 * 4)
            hipLaunchKernelGGL((k_gn_group<DT, V, 256, 16 / V>), grid, dim3(256), 0, s, *d);
        else if (d->rows * (d->C / d->groups) <= 1024 * 16)
            hipLaunchKernelGGL((k_gn_group<DT, V, 1024, 16 / V>), grid, dim3(1024), 0, s, *d);
        else
            hipLaunchKernelGGL((k_gn_group<DT, V, 1024, 0>), grid, dim3(1024), 0, s, *d);
    }
    else {
        hipLaunchKernelGGL((k_gn_stats<DT, V>), dim3(d->chunks, d->nb), dim3(TH), 0, s, *d);
        err = hipGetLastError();
        if (err == hipSuccess && d->stats) {
            hipLaunchKernelGGL(k_gn_sums, dim3((d->groups + 3) / 4, d->nb), dim3(256), 0, s, *d);
            err = hipGetLastError();
        }
        if (err != hipSuccess)
            return err;
        hipLaunchKernelGGL((k_gn_apply<DT, V>), dim3(d->chunks / 2, d->nb), dim3(TH),
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
    if (!ws || ws_bytes < part_bytes(d))
        d->chunks = 1;
    d->part = (float *)ws;
    /* A launch of its own for the sums where every workgroup would read more
     * than 64 KiB of them: 3 batches of 5184 rows of 256 halves, 32 groups 17.7
     * us and 19.7, 82944 rows of 256 floats, 8 groups 41.3 and 40.0. */
    d->stats = d->chunks > 1 && (long)d->chunks * d->groups > 4096
                   ? (char *)ws + 16 * (size_t)d->nb * d->groups * d->chunks
                   : NULL;
    return d->dt == DT_F32   ? run_dt<DT_F32>(d, (hipStream_t)stream)
           : d->dt == DT_F16 ? run_dt<DT_F16>(d, (hipStream_t)stream)
                             : run_dt<DT_BF16>(d, (hipStream_t)stream);
}
