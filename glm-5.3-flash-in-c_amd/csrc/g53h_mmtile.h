/* g53h_mmtile.h - tiles of matrix products that stream their operands through LDS, for the products of sorted rows
 * (g53h_emm.hip) and of microscaled matrices (g53h_mx4.hip).
 *
 * A workgroup of WR x WC waves owns a tile of BM x BN results; each of its waves MT x NT tiles of 16 x 16. It takes the
 * summed dimension in chunks: 128 bytes of every operand row where a row holds the summed elements side by side
 * ("along": x and W forward), or as many of its rows where they lie across ("across": W for the rows' gradient, both
 * operands of the matrices'). Either way a chunk is 128 bytes for each of the tile's rows or columns, and moves in
 * pieces of 16 bytes, 64 a wave and instruction, straight to LDS (global_load_lds) into a ring of slots. The loads are
 * inline assembly, and waits count them by hand: the compiler would wait for every load to LDS before any LDS read.
 *
 * LDS places. Along: row r is 128 bytes, piece u of it at u ^ (r % 8), so the 16 rows that a fragment read meets lie in
 * all banks. Across: a row of the chunk holds the tile's columns, piece u at u ^ f(k): the rows that a transposing read
 * (ds_read_b64_tr_b16: 4 rows x 16 columns for 16 lanes) or a read of fp32 columns meets in one go lie in all banks.
 */
#ifndef G53H_MMTILE_H
#define G53H_MMTILE_H

#include <hip/hip_runtime.h>
#include <type_traits>

#include "g53h.h"
#include "g53h_elem.h"

typedef short g53_v4s __attribute__((ext_vector_type(4)));
typedef g53_v4s __attribute__((address_space(3))) *G53LdsTr;

static __device__ const g53_v4w g53_nothing = {0, 0, 0, 0};     /* what a load behind an operand's end reads */

/* A value every lane reads alike from memory that no kernel of this launch writes: a scalar load. */
template <class V> __device__ __forceinline__ V g53_uniform_load(const V *p)
{
    return *(const __attribute__((address_space(4))) V *)(uintptr_t)p;
}

/* 16 bytes per lane from p to LDS byte lds + 16 * lane. M0 holds the LDS address and is written ahead of the load. */
__device__ __forceinline__ void g53_to_lds(const uint8_t *p, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}
/* At most n loads of the wave are on their way behind this; then every wave of the workgroup gets here. */
template <int n> __device__ __forceinline__ void g53_loads_left()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}
__device__ __forceinline__ void g53_meet()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

/* p / topk for a pair number p (below 2^31) by a product: mul = ceil(2^(31 + l) / topk), l = the bits of topk - 1. */
struct G53Div {
    uint32_t mul;
    int l;
};
static inline G53Div g53_div_of(int d)
{
    int l = 0;
    while ((1 << l) < d) l++;
    return {(uint32_t)(((1ull << (31 + l)) + (unsigned)d - 1) / (unsigned)d), l};
}
__device__ __forceinline__ int g53_div(int p, G53Div d) { return (int)(__umulhi((uint32_t)p << 1, d.mul) >> d.l); }

/* Rows [first, last) of expert e: the tile `item / across` in the experts' order, tiles of TM rows; n the tile across.
 * Items are dealt to the 8 dies in runs of up to 16, so that a die's cache serves a tile's operands to the others of the
 * run (4096 x 4096, 64 experts, 4096 tokens of top-8: runs of 8 1151 us, of 16 1096, of 32 1125). Within an expert eight tiles of rows go with each tile across. False
 * where the launch has no item for the workgroup. */
struct G53Item {
    int e, first, last, n;
};
template <typename I> __device__ __forceinline__ I g53_deal(I wg, I total)
{
    if (total >= 256) return (wg >> 7 << 7) + (wg & 7) * 16 + (wg >> 3 & 15);       /* runs of 16 */
    const I run = total >= 16 ? total / 8 : 1, i = wg >> 3;
    return ((i / run) * 8 + (wg & 7)) * run + i % run;
}
/* The workgroups that cover `total` items so dealt, or fewer. */
static inline long g53_deal_wgs(long total) { return (total + 7) / 8 * 8 + (total < 8 ? 8 : total < 256 ? (total + 7) / 8 * 8 : 256); }
/* Item `in` of tiles x across: eight tiles go with each tile across. */
template <typename I> __device__ __forceinline__ void g53_eight(I in, int tiles, int across, int &t, int &n)
{
    const I eight = (I)8 * across;
    const int g = (int)(in / eight), in_g = (int)(in - g * eight), of = tiles - 8 * g < 8 ? tiles - 8 * g : 8;
    t = 8 * g + in_g % of;
    n = in_g / of;
}
__device__ __forceinline__ bool g53_tile_item(const int *__restrict__ offsets, int NE, int TM, int across, long wg,
                                              G53Item &it)
{
    const int lane = threadIdx.x & 63, per = (NE + 63) / 64, e0 = lane * per;
    int n = 0, from = e0 < NE ? offsets[e0] : 0;
    for (int i = 0, at = from; i < per; i++)
        if (e0 + i < NE) {
            const int to = offsets[e0 + i + 1];
            n += (int)(((unsigned)(to - at) + TM - 1) / TM);
            at = to;
        }
    int incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    const long total = (long)__builtin_amdgcn_readlane(incl, 63) * across;
    const long item = g53_deal(wg, total);
    if (item >= total) return false;
    const unsigned long long in = __ballot((long)incl * across > item);
    const int l = __builtin_ctzll(in);
    long left = item - (long)__builtin_amdgcn_readlane(incl - n, l) * across;
    int first = __builtin_amdgcn_readlane(from, l), last, e = l * per, tiles;
    for (;; e++) {                      /* lane l's experts: one of them holds the item */
        last = g53_uniform_load(offsets + e + 1);
        tiles = (int)(((unsigned)(last - first) + TM - 1) / TM);
        if (left < (long)tiles * across) break;
        left -= (long)tiles * across;
        first = last;
    }
    int t, n_;
    g53_eight(left, tiles, across, t, n_);
    it.n = __builtin_amdgcn_readfirstlane(n_);
    it.e = __builtin_amdgcn_readfirstlane(e);
    it.first = __builtin_amdgcn_readfirstlane(first + t * TM);
    it.last = __builtin_amdgcn_readfirstlane(last - it.first > TM ? it.first + TM : last);
    return true;
}

/* Where a lane's 16 bytes of a chunk come from, how many bytes its row has from there on (0 and less: none), and whether
 * the row is there at all; the address is that of a row in any case. */
struct G53Piece {
    const uint8_t *p;
    int n;
    bool row;
};
/* Pieces through registers, at any alignment of their elements (of type E). All of a thread's are asked for together and
 * looked at when they are put down: one that meets its row's end is the row's last 16 bytes, moved down by `by` then
 * (16: nothing is there, zeros). Rows of less than 16 bytes go by elements. */
__device__ __forceinline__ void g53_take(g53_v4w &o, int &by, const G53Piece &s)
{
    const int back = s.n >= 16 ? 0 : 16 - s.n;
    o = ((const G53v4w_any *)(s.p - back))->v;
    by = s.row && back < 16 ? back : 16;
}
template <typename E> __device__ __forceinline__ void g53_take_short(g53_v4w &o, int &by, const G53Piece &s)
{
    const E *p = (const E *)s.p;
    constexpr int N = 16 / sizeof(E);
    const int n = s.row ? s.n / (int)sizeof(E) : 0;
    E v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = i < n ? p[i] : (E)0.0f;
    __builtin_memcpy(&o, v, 16);
    by = 0;
}
template <typename E> __device__ __forceinline__ g53_v4w g53_moved(const g53_v4w &v, int by)
{
    unsigned d[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = by & 8 ? (i < 2 ? d[i + 2] : 0u) : d[i];
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = by & 4 ? (i < 3 ? d[i + 1] : 0u) : d[i];
    if (sizeof(E) == 2)
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = by & 2 ? __builtin_amdgcn_alignbyte(i < 3 ? d[i + 1] : 0u, d[i], 2) : d[i];
    return (g53_v4w){by & 16 ? 0u : d[0], by & 16 ? 0u : d[1], by & 16 ? 0u : d[2], by & 16 ? 0u : d[3]};
}

/* The 16-bit type of the products and the planes of a value. fp32 enters as three bf16 planes, each the rounded rest of
 * those before it: with 8 bits a plane and at most half a step left by each, the three hold every bit of the value
 * (above 2^-109; and values that round past bf16's largest, from 3.396e38, count as infinite). Of the nine products
 * of two values' planes six are taken. The planes of a value in [1, 2) are at most 2^-8 and 2^-17, so the others are below
 * 2^-24 of the values' product together, fp32's own rounding of one (2^-24.01 for 0x1.00ff8p0 by itself, 2^-28 in the mean of
 * random values, of either sign). */
template <typename E> struct G53Mm;
template <> struct G53Mm<float> { typedef g53_v8b V; static constexpr int P = 3; };
template <> struct G53Mm<g53_bf16> { typedef g53_v8b V; static constexpr int P = 1; };
template <> struct G53Mm<g53_f16> { typedef g53_v8h V; static constexpr int P = 1; };

__device__ __forceinline__ g53_v4f g53_mm(g53_v8b a, g53_v8b b, g53_v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ g53_v4f g53_mm(g53_v8h a, g53_v8h b, g53_v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename E> struct G53Frag { typename G53Mm<E>::V v[G53Mm<E>::P]; };

__device__ __forceinline__ void g53_planes(G53Frag<float> &o, const float (&v)[8])
{
    typedef float F2 __attribute__((ext_vector_type(2)));
    typedef g53_bf16 B2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int p = 0; p < 3; p++) {                       /* two at a time: one conversion */
            const B2 h = __builtin_convertvector((F2){a, b}, B2);
            o.v[p][2 * i] = h[0];
            o.v[p][2 * i + 1] = h[1];
            if (p == 2) break;
            const unsigned u = __builtin_bit_cast(unsigned, h);
            a -= __builtin_bit_cast(float, u << 16);        /* exact */
            b -= __builtin_bit_cast(float, u & 0xffff0000u);
        }
    }
}
template <typename E> __device__ __forceinline__ g53_v4f g53_mm(const G53Frag<E> &a, const G53Frag<E> &b, g53_v4f c)
{
    if constexpr (G53Mm<E>::P == 3) {
        c = g53_mm(a.v[2], b.v[0], c);
        c = g53_mm(a.v[1], b.v[1], c);
        c = g53_mm(a.v[0], b.v[2], c);
        c = g53_mm(a.v[1], b.v[0], c);
        c = g53_mm(a.v[0], b.v[1], c);
        return g53_mm(a.v[0], b.v[0], c);
    } else {
        return g53_mm(a.v[0], b.v[0], c);
    }
}

/* Fragments of 32 summed elements (lane (m, q) = (lane % 16, lane / 16): row m, elements 8 q .. 8 q + 7) from a chunk
 * at LDS address `at`, whose rows start at row0 (a multiple of 16), tile t of 16 rows, every STRIDE-th, step j of 32 elements. */
template <typename E, int STRIDE = 1> struct G53Along {
    int at[2];
    __device__ __forceinline__ void setup(int row0)
    {
        const int m = threadIdx.x & 15, q = threadIdx.x >> 4 & 3;
        const int u = sizeof(E) == 4 ? 2 * q : q;
        at[0] = (row0 + m) * 128 + ((u ^ (m & 7)) << 4);
        at[1] = sizeof(E) == 4 ? (row0 + m) * 128 + (((u + 1) ^ (m & 7)) << 4) : at[0] ^ 64;
    }
    __device__ __forceinline__ void read(G53Frag<E> &o, const uint8_t *lds, int t, int j) const
    {
        if constexpr (sizeof(E) == 4) {
            const g53_v4f a = *(const g53_v4f *)(lds + at[0] + t * STRIDE * 2048), b = *(const g53_v4f *)(lds + at[1] + t * STRIDE * 2048);
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
            g53_planes(o, v);
        } else {
            o.v[0] = *(const typename G53Mm<E>::V *)(lds + at[j] + t * STRIDE * 2048);
        }
    }
};
/* The same from a chunk of rows of R columns each, whose columns start at col0: NT tiles of 16. */
template <typename E, int R, int NT, int STRIDE = 1> struct G53Across {
    static constexpr int RB = R * sizeof(E), U = RB / 16;         /* bytes and pieces of a row */
    int at0;
    static __device__ __forceinline__ int place(int k)
    {
        return (sizeof(E) == 4 ? 4 * (k >> 3 & 3) : 2 * ((k & 3) | (k >> 3 & 1) << 2)) & (U - 1);
    }
    /* Of rows k, k + step, k + 2 step, ... how many until places repeat. */
    template <int step> static constexpr int turns()
    {
        constexpr int period = sizeof(E) == 4 ? 32 : 16;
        static_assert(step % 8 == 0, "rows of eight");
        return step % period ? period / step : 1;
    }
    /* A tile's columns are other bits of a place than col0's: one address, the others by exclusive or. */
    __device__ __forceinline__ void setup(int col0)
    {
        const int m = threadIdx.x & 15, q = threadIdx.x >> 4 & 3;
        const int k = sizeof(E) == 4 ? 8 * q : 8 * q + (m >> 2);
        const int u = sizeof(E) == 4 ? (col0 + m) >> 2 : (col0 >> 3) + (m >> 1 & 1);
        at0 = k * RB + ((u ^ place(k)) << 4) + (sizeof(E) == 4 ? (m & 3) * 4 : (m & 1) * 8);
    }
    __device__ __forceinline__ void read(G53Frag<E> &o, const uint8_t *lds, int t, int j) const
    {
        const int at = at0 ^ (16 * STRIDE * t * (int)sizeof(E));
        if constexpr (sizeof(E) == 4) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = *(const float *)(lds + at + i * RB);
            g53_planes(o, v);
        } else {
            const g53_v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((G53LdsTr)(lds + at + j * 32 * RB));
            const g53_v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((G53LdsTr)(lds + at + (j * 32 + 4) * RB));
            o.v[0] = __builtin_bit_cast(typename G53Mm<E>::V, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

/* A wave's MT x n tiles to memory, each value rounded once. They go through LDS (buf: 16 MT x 16 n elements of the wave's own)
 * and leave as pieces of 16 bytes, whole rows of the wave's columns: a store of the sums as they lie would leave 64 bytes of
 * each of 16 rows. (Rows of less than 128 bytes go as they lie: one token 15.8 us against 18.4.) The loop over pieces is not unrolled whole: small calls wait for every instruction of it to be fetched.
 * out: the first row's first column; tile i is 16 STRIDE i rows on. ld: elements from row to row; rows, cols: how many there are. */
template <typename O, int STRIDE, int MT, int n>
__device__ __forceinline__ void g53_leave(uint8_t *buf, O *out, long ld, const g53_v4f (&v)[MT][n], int rows, int cols)
{
    constexpr int RB = n * 16 * sizeof(O), PR = RB / 16, RI = 64 / PR, EP = 16 / sizeof(O), SW = (PR < 8 ? PR : 8) - 1;
    typedef O V4 __attribute__((ext_vector_type(4)));
    if constexpr (RB < 128) {
        struct __attribute__((packed, aligned(2))) Any4 { V4 v; };
        const int m = threadIdx.x & 15, q = threadIdx.x >> 4 & 3;
#pragma unroll
        for (int i = 0; i < MT; i++) {
            if (16 * STRIDE * i + m >= rows) continue;
#pragma unroll
            for (int t = 0; t < n; t++) {
                O *to = out + (16 * STRIDE * i + m) * ld + 16 * t + 4 * q;
                V4 o;
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = (O)v[i][t][k];
                const int left = cols - 16 * t - 4 * q;
                if (left >= 4) ((Any4 *)to)->v = o;
                else
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (k < left) to[k] = o[k];
            }
        }
        return;
    } else {
    typedef O VP __attribute__((ext_vector_type(EP)));
    struct __attribute__((packed, aligned(2))) Any { VP v; };
    static_assert(16 * MT % RI == 0, "whole rounds of rows");
    const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < n; t++) {
            const int b = (16 * t + 4 * q) * (int)sizeof(O);
            V4 o;
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = (O)v[i][t][k];
            *(V4 *)(buf + (16 * i + m) * RB + (((b >> 4) ^ (m & SW)) << 4) + (b & 15)) = o;
        }
    const int p = lane % PR, left = cols - p * EP;
#pragma unroll 4
    for (int k = 0; k < 16 * MT / RI; k++) {
        const int r = k * RI + lane / PR, at = (r >> 4) * (16 * STRIDE) + (r & 15);
        const VP o = *(const VP *)(buf + r * RB + ((p ^ (r & SW)) << 4));
        O *to = out + at * ld + p * EP;
        if (at >= rows) continue;
        if (left >= EP) ((Any *)to)->v = o;
        else
            for (int i = 0; i < left; i++) to[i] = ((const O *)(buf + r * RB + ((p ^ (r & SW)) << 4)))[i];
    }
    }
}
/* The same for sums that may be added to what is there: they pass LDS (16 MT x 16 n fp32) as they are, are added in fp32 and
 * rounded then, to fp32 or to O. Whole pieces go past the caches: these results are many, and whoever reads them does so
 * much later (4.3 GB 1472 us against 1589). */
template <typename O, int STRIDE, int MT, int n>
__device__ __forceinline__ void g53_leave_sums(uint8_t *buf, void *out, long first, long ld, const g53_v4f (&v)[MT][n], int rows, int cols,
                                               bool f32, bool old)
{
    constexpr int RB = n * 64;
    const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < n; t++) *(g53_v4f *)(buf + (16 * i + m) * RB + (((4 * t + q) ^ (m & 7)) << 4)) = v[i][t];
    auto all = [&](auto *base) {
        typedef typename std::remove_pointer<decltype(base)>::type T;
        constexpr int EP = 16 / sizeof(T), PR = n * 16 / EP, RI = 64 / PR;      /* a lane's 16 bytes of result */
        typedef T V __attribute__((ext_vector_type(EP)));
        static_assert(16 * MT % RI == 0 && (STRIDE == 1 || RI <= 16), "whole rounds of rows");
        const int p = lane % PR, left = cols - EP * p, r0 = lane / PR;
        T *row = base + first + r0 * ld + EP * p;
        if (rows >= 16 * (STRIDE * (MT - 1) + 1) && cols >= 16 * n && !old && !(((uintptr_t)base | (first | ld) * sizeof(T)) & 15)) {
#pragma unroll 4
            for (int k = 0; k < 16 * MT / RI; k++) {        /* all there, in whole pieces */
                const int r = k * RI + r0;
                V w;
#pragma unroll
                for (int h = 0; h < EP / 4; h++) {
                    const g53_v4f part = *(const g53_v4f *)(buf + r * RB + (((EP / 4 * p + h) ^ (r & 7)) << 4));
#pragma unroll
                    for (int i = 0; i < 4; i++) w[4 * h + i] = (T)part[i];
                }
                __builtin_nontemporal_store(w, (V *)row);
                row += (RI % 16 == 0 ? RI * STRIDE : (k + 1) * RI % 16 ? RI : RI + 16 * (STRIDE - 1)) * ld;
            }
            return;
        }
#pragma unroll 1
        for (int k = 0; k < 16 * MT / RI; k++) {
            const int r = k * RI + r0, at = (r >> 4) * (16 * STRIDE) + (r & 15);
            if (at >= rows || left <= 0) continue;
            row = base + first + at * ld + EP * p;
#pragma unroll
            for (int i = 0; i < EP; i++) {
                const int c = EP * p + i;                   /* its fp32 in LDS */
                const float o = *(const float *)(buf + r * RB + (((c >> 2) ^ (r & 7)) << 4) + (c & 3) * 4);
                if (i < left) row[i] = (T)(old ? o + (float)row[i] : o);
            }
        }
    };
    if (f32) all((float *)out);
    else all((O *)out);
}

/* The clamped SwiGLU, as g53h_swiglu's, for a result of type O. One of 16 bits, whose half step is 2^-11 of a value and more,
 * takes the hardware's exponential and reciprocal: they take a quarter of the time, and at the end of a tile nothing covers it.
 * Off by some 2^-20 together, and |gate| 2^-24 more where the gate is negative (its product with log2 e is rounded); 0 where the
 * exponential lies below 2^-126, gates of -87.4 and less. */
template <typename O> __device__ __forceinline__ float g53_swiglu1(float g, float u, float limit)
{
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
    if constexpr (sizeof(O) == 2) {
        const float e = __expf(-fabsf(g));                  /* no overflow, so no reciprocal below the normal range */
        return g * ((g >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e)) * u;
    } else {
        return g / (1.0f + expf(-g)) * u;
    }
}

#endif /* G53H_MMTILE_H */
