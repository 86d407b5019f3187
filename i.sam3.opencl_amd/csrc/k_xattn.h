/* SPDX-License-Identifier: Unlicense
 *
 * What the kernels of cross_attend share: element types, the MFMA steps, the
 * layout of K and V in LDS and the copies into it, the order of the work.
 */
#ifndef K_XATTN_H
#define K_XATTN_H

#include "k_common.h"

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct yes {
    static constexpr bool value = true;
};
struct no {
    static constexpr bool value = false;
};

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

/* 16 bytes of a row at column byte cb: whole, or element by element, with
 * zeros from column hd on. */
template <int DT, bool VEC>
__device__ __forceinline__ u32x4 row16(const char *p, int cb, int hdb)
{
    constexpr int S = xt<DT>::size;
    u32x4 v = {0, 0, 0, 0};

    if (cb >= hdb)
        return v;
    if (VEC)
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

/* One 16-byte step of S^T = K Q^T. */
template <int DT> __device__ __forceinline__ f32x16 k_step(u32x4 k, u32x4 q, f32x16 s)
{
    if constexpr (DT == DT_F32) {
        const f32x4 kx = __builtin_bit_cast(f32x4, k), qx = __builtin_bit_cast(f32x4, q);

#pragma unroll
        for (int e = 0; e < 4; e++)
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(kx[e], qx[e], s, 0, 0, 0);
        return s;
    }
    else
        return mfma16<DT>(k, q, s);
}

/* Column c of output row p. */
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

/* Sixteen zeros: what stands for columns past the head width. */
__device__ const u32x4 xattn_zeros = {0, 0, 0, 0};

/* Layout of a tile's rows (RB bytes) in LDS. A copy fills 1 KiB, RPK rows; PAD
 * bytes follow each. Chunk c (16 bytes) of row r stands in slot c ^ swz(r) of
 * its row. LDS serves 256 bytes at once: K is read as one chunk of 32 rows,
 * and 16 rows in turn take 16 different slots; V is read as 64 bytes of four
 * rows (transposed, 16 bits) or 128 bytes of two rows four apart (floats),
 * which take different quarters or halves. swz depends on r % RPK alone, and
 * on few bits, so that an address is one of few registers and a constant. */
template <int RB> struct row_k {
    static constexpr int RPK = 1024 / RB;
    static constexpr int PAD = RB == 64 ? 0 : RB <= 256 ? 64 : RB == 512 ? 32 : 16;
    __device__ static __forceinline__ int swz(int r)
    {
        return RB == 64 ? r >> 2 & 3 : RB == 128 ? r >> 1 & 3 : RB == 256 ? r & 3 : RB == 512 ? r & 1 : 0;
    }
    __device__ static __forceinline__ int at(int r)
    {
        return r / RPK * (1024 + PAD) + r % RPK * RB;
    }
};
template <int RB, int DT> struct row_v {
    static constexpr int RPK = 1024 / RB;
    static constexpr int PAD = DT == DT_F32 ? (RB == 256 ? 128 : RB == 512 ? 64 : RB == 1024 ? 32 : 0)
                               : RB == 512 ? 128 : 0;
    __device__ static __forceinline__ int swz(int r)
    {
        return DT == DT_F32 ? 0 : RB == 128 ? (r >> 1 & 1) << 2 : RB == 256 ? (r & 3) << 2 : RB == 512 ? (r & 1) << 2 : 0;
    }
    __device__ static __forceinline__ int at(int r)
    {
        return r / RPK * (1024 + PAD) + r % RPK * RB;
    }
};

/* Lanes read what others of their wave have written to LDS: served in order,
 * which the compiler has to keep. */
__device__ __forceinline__ void wave_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

/* The same copy as g2lds16 from an address of each lane's own. */
__device__ __forceinline__ void g2lds16_at(const void *src, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds), "v"(src)
                 : "memory", "m0");
}

/* Waits until at most N of this wave's copies (the last issued) are under
 * way, and for its LDS accesses, then for the workgroup. */
template <int N> __device__ __forceinline__ void copies_and_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\t"
                 "s_barrier"
                 :
                 : "n"(N)
                 : "memory");
}

/* The work of this workgroup, of groups x members: the members of a group share
 * memory (a unit's keys, or the rows of all heads) and an XCD (workgroup index
 * mod 8), whose L2 then holds it. XCDs take every eighth group, so that long and
 * short sequences spread over them, or, where that would leave some with less, a
 * contiguous eighth of the items each. us against contiguous eighths always:
 * step of 16 sequences over up to 8192 keys 76.6 and 79.5, ragged batch of 4 x
 * 447 rows over 1500 keys 19.9 and 21.4, 8 x 5184 rows over 37 keys 11.4 and
 * 12.3. item_grid: workgroups of the launch. */
__device__ __host__ __forceinline__ bool every_eighth(unsigned groups)
{
    return groups % 8 == 0 || groups >= 64;
}

static unsigned item_grid(unsigned groups, unsigned members)
{
    return every_eighth(groups) ? (groups + 7) / 8 * 8 * members
                                : (groups * members + 7) / 8 * 8;
}

__device__ __forceinline__ bool item_of(unsigned groups, unsigned members, unsigned *group,
                                        unsigned *member)
{
    const unsigned x = blockIdx.x & 7, j = blockIdx.x >> 3;

    if (every_eighth(groups)) {
        const unsigned i = j / members;

        *group = 8 * i + x;
        *member = j - i * members;
        return *group < groups;
    }
    const unsigned item = x * ((groups * members + 7) / 8) + j;

    *group = item / members;
    *member = item - *group * members;
    return j < (groups * members + 7) / 8 && *group < groups;
}

/* Columns c to c + 31 of an output row: this lane's half (h) of the sums in o,
 * times inv. */
template <int DT, bool VEC>
__device__ __forceinline__ void put_block(char *op, int c, int hd, int h, const f32x16 &o, float inv)
{
#pragma unroll
    for (int q = 0; q < 4; q += 2, c += 16) {
        float x[8];

#pragma unroll
        for (int e = 0; e < 8; e++)
            x[e] = o[4 * q + e] * inv;
        if constexpr (!VEC) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int ce = c + 8 * (e / 4) + 4 * h + e % 4;

                if (ce < hd)
                    put_elem<DT>(op, ce, x[e]);
            }
        }
        else if constexpr (DT == DT_F32) {
            if (c + 4 * h < hd)
                *(f32x4 *)(op + 4 * (c + 4 * h)) = f32x4{x[0], x[1], x[2], x[3]};
            if (c + 8 + 4 * h < hd)
                *(f32x4 *)(op + 4 * (c + 8 + 4 * h)) = f32x4{x[4], x[5], x[6], x[7]};
        }
        else {
            /* Lanes 32 apart exchange halves: 8 columns in a row each. */
            const auto u = __builtin_amdgcn_permlane32_swap(
                pack2<DT>(x[0], x[1]), pack2<DT>(x[4], x[5]), false, false);
            const auto v = __builtin_amdgcn_permlane32_swap(
                pack2<DT>(x[2], x[3]), pack2<DT>(x[6], x[7]), false, false);

            if (c + 8 * h < hd)
                *(u32x4 *)(op + 2 * (c + 8 * h)) =
                    u32x4{(uint32_t)u[0], (uint32_t)v[0], (uint32_t)u[1], (uint32_t)v[1]};
        }
    }
}

#endif /* K_XATTN_H */
