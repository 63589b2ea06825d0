/* g53h_elem.h - elements of the operators that take several types (G53H_F32, G53H_BF16, G53H_F16):
 * eight of them at a time to and from fp32 registers. Addresses need the alignment of one element
 * only: gfx950 loads and stores 16 bytes at any address, and rows of odd length start anywhere.
 */
#ifndef G53H_ELEM_H
#define G53H_ELEM_H

#include <hip/hip_runtime.h>

#include "g53h.h"

typedef __bf16 g53_bf16;
typedef _Float16 g53_f16;
typedef float g53_v4f __attribute__((ext_vector_type(4)));
typedef unsigned int g53_v4w __attribute__((ext_vector_type(4)));
typedef g53_bf16 g53_v8b __attribute__((ext_vector_type(8)));
typedef g53_f16 g53_v8h __attribute__((ext_vector_type(8)));

/* The same vectors at any 2-byte address. */
struct __attribute__((packed, aligned(2))) G53v4w_any { g53_v4w v; };
struct __attribute__((packed, aligned(2))) G53v8b_any { g53_v8b v; };
struct __attribute__((packed, aligned(2))) G53v8h_any { g53_v8h v; };
struct __attribute__((packed, aligned(4))) G53v4f_any { g53_v4f v; };

/* Bytes of an element of type dt, 0 if dt is none of the types. */
static inline int g53_elem_bytes(int dt) { return dt == G53H_F32 ? 4 : (dt == G53H_BF16 || dt == G53H_F16 ? 2 : 0); }

__device__ __forceinline__ void g53_load8(float (&o)[8], const float *p)
{
    const g53_v4f a = ((const G53v4f_any *)p)[0].v, b = ((const G53v4f_any *)p)[1].v;
#pragma unroll
    for (int i = 0; i < 4; i++) { o[i] = a[i]; o[4 + i] = b[i]; }
}
__device__ __forceinline__ void g53_load8(float (&o)[8], const g53_bf16 *p)
{
    const g53_v8b a = ((const G53v8b_any *)p)->v;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = (float)a[i];
}
__device__ __forceinline__ void g53_load8(float (&o)[8], const g53_f16 *p)
{
    const g53_v8h a = ((const G53v8h_any *)p)->v;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = (float)a[i];
}
/* Stores round to the nearest value of the type, ties to even: half a step each. */
__device__ __forceinline__ void g53_store8(float *p, const float (&v)[8])
{
    g53_v4f a, b;
#pragma unroll
    for (int i = 0; i < 4; i++) { a[i] = v[i]; b[i] = v[4 + i]; }
    ((G53v4f_any *)p)[0].v = a;
    ((G53v4f_any *)p)[1].v = b;
}
__device__ __forceinline__ void g53_store8(g53_bf16 *p, const float (&v)[8])
{
    g53_v8b a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = (g53_bf16)v[i];
    ((G53v8b_any *)p)->v = a;
}
__device__ __forceinline__ void g53_store8(g53_f16 *p, const float (&v)[8])
{
    g53_v8h a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = (g53_f16)v[i];
    ((G53v8h_any *)p)->v = a;
}

/* Elements c .. c + 7 of a row of n, zeros behind its end: a lane whose eight all lie there reads nothing, one that meets
 * the end reads the last element in their place, without a branch. */
template <typename T> __device__ __forceinline__ void g53_load8_to(float (&o)[8], const T *row, int c, int n)
{
    if (c + 8 <= n) {
        g53_load8(o, row + c);
    } else if (c >= n) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = 0.0f;
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = row[c + i < n ? c + i : n - 1];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = c + i < n ? (float)v[i] : 0.0f;
    }
}
template <typename T> __device__ __forceinline__ void g53_store8_to(T *row, const float (&v)[8], int c, int n)
{
    if (c + 8 <= n) {
        g53_store8(row + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (c + i < n) row[c + i] = (T)v[i];
    }
}

/* The same eight as they lie, for loads that are waited for later. */
template <typename T> struct G53Raw8 { T v __attribute__((ext_vector_type(8))); };
template <typename T> __device__ __forceinline__ void g53_raw8_to(G53Raw8<T> &o, const T *row, int c, int n)
{
    typedef T V8 __attribute__((ext_vector_type(8)));
    struct __attribute__((packed, aligned(2))) Any { V8 v; };
    if (c + 8 <= n) {
        o.v = ((const Any *)(row + c))->v;
    } else if (c >= n) {
#pragma unroll
        for (int i = 0; i < 8; i++) o.v[i] = (T)0.0f;
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = row[c + i < n ? c + i : n - 1];
#pragma unroll
        for (int i = 0; i < 8; i++) o.v[i] = c + i < n ? v[i] : (T)0.0f;
    }
}

/* The same for rows that are read once: they need not stay in the caches. */
template <typename T> __device__ __forceinline__ void g53_raw8_once_to(G53Raw8<T> &o, const T *row, int c, int n)
{
    if (c + 8 <= n && !((uintptr_t)(row + c) & 15)) {
        typedef T V8 __attribute__((ext_vector_type(8)));
        o.v = __builtin_nontemporal_load((const V8 *)(row + c));
    } else {
        g53_raw8_to(o, row, c, n);
    }
}

/* The loads into o are waited for here. Stores count as loads do, so a wait behind them would be for them too. */
template <typename T> __device__ __forceinline__ void g53_arrived(G53Raw8<T> &o)
{
    typedef unsigned int Words __attribute__((ext_vector_type(sizeof(o.v) / 4)));
    Words w = __builtin_bit_cast(Words, o.v);
    asm volatile("" : "+v"(w));
    o.v = __builtin_bit_cast(decltype(o.v), w);
}

/* v of the lane that DPP control ctrl names, inside each row of 16 lanes. */
template <int ctrl> __device__ __forceinline__ float g53_dpp(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true));
}

/* The sum of v over the 64 lanes of a wave, the same bits in every lane: pairs, quads and halves of a row of 16 lanes by
 * DPP, rows and halves of the wave by register swaps, no trip through LDS. */
__device__ __forceinline__ float g53_wave_sum(float v)
{
    v += g53_dpp<0xb1>(v);              /* lane ^ 1 */
    v += g53_dpp<0x4e>(v);              /* lane ^ 2 */
    v += g53_dpp<0x141>(v);             /* 7 - lane: the other quad of eight */
    v += g53_dpp<0x140>(v);             /* 15 - lane: the other eight of the row */
    typedef unsigned int V2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int half = 0; half < 2; half++) {          /* the other row of two, then the other two rows */
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const V2 p = half ? __builtin_amdgcn_permlane32_swap(u, u, false, false)
                          : __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const unsigned a = p[0], b = p[1];          /* a bit cast of a vector's element takes element 0 */
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    return v;
}

/* Run a kernel template over the element type that dt names: BODY sees it as E. */
#define G53_BY_TYPE(dt, BODY)                                             \
    do {                                                                  \
        if ((dt) == G53H_F32) { typedef float E; BODY; }                  \
        else if ((dt) == G53H_BF16) { typedef g53_bf16 E; BODY; }         \
        else { typedef g53_f16 E; BODY; }                                 \
    } while (0)

#endif /* G53H_ELEM_H */
