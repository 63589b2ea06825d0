/* g53h_w4.hip - products of a few tokens with matrices of 4-bit levels and group scales, of one
 * matrix (g53h_mm_w4) or of the matrix of each sorted row's expert (g53h_sorted_mm_w4):
 *
 *     y[t][r] = sum over groups g of  s[r][g] * sum over c in g of (q[r][c] - z[r][g]) x[t][c]
 *
 * Levels go to the matrix cores as whole numbers, exact in bf16 and fp16, and the scale joins a group's
 * sum. With fp32 and fp16 activations they go as q - z. A sum of (16 + q) x, which takes less work to
 * form, is many times the result where x has a mean or one large value, and its roundings stay when
 * (16 + z) X comes off, X the group's sum of x: fp32 x = N(1, 1) by weights around 0, 4096 columns, 3e-6
 * of the result's norm off against 1e-7 of q - z and 4e-7 of a plain fp32 sum; 2^13 in one column
 * 1e-4 of the rows in which its level is z, against 1e-7. (65536 x 4096 by 5 fp16 tokens 29.5 us against
 * 28.8, 16384 x 4096 by one in fp32 11.3 against 9.8.) fp16: one conversion takes two levels, as e4m3 codes
 * of q 2^-9, and one packed subtraction z off them. fp32 activations enter as three bf16 planes whose sum
 * is the value exactly (8 + 8 + 8 mantissa bits, by truncation), and their levels, since bf16 has no
 * packed subtraction, as four bytes less z, then fp32, whose upper halves are bf16. With bf16 activations
 * levels go as q and z X comes off, X by one product with ones that all row tiles share: roundings are
 * those of
 * sums of (q + z) s |x|, 2^-24 each, below a result that keeps 2^-9 of itself (with 2^13 in one column 1
 * of 150 results is not the nearest bf16, with 16 + q 1 of 70; q - z as with fp32: 65536 x 4096 by one
 * token 33.4 us against 26.7). Products are exact and sums fp32.
 *
 * A wave owns R tiles of 16 rows and NT tiles of 16 tokens over a part of the columns and steps by 128
 * columns: one 16-byte load per lane and row tile (16 rows x 64 bytes, or 8 rows x whole lines of 128).
 * Where a chunk of 128 columns lies in one group, each of its four products takes 8 columns of every
 * lane quarter's 32; in groups of 32, 64 or 96 the registers are turned so that a product covers 32
 * columns in a row and groups end between products (v_permlane32_swap and v_permlane16_swap exchange the
 * lanes' quarters with the four registers). The NW waves of a workgroup split the columns and add up
 * through LDS, which also holds the activations, turned into planes once a workgroup, except for small
 * matrices, whose waves each load theirs.
 *
 * By few tokens the levels' bytes bound it: 65536 x 4096 by 5 fp16 tokens 29.5 us, 4.8 TB/s (a plain
 * read stream of as many bytes: 23 to 26); eight gate/up matrices of 4096 x 4096 by one token 16.5 us,
 * 4.2 TB/s with a launch and the search of a row's expert in it. Matrices of 10 to 40 MB leave part of
 * the card idle at their start and end (9000 x 8192 by 5 tokens 18.1 us, 2.1 TB/s). Small ones are a
 * launch and three trips to memory (4096 x 2048 by one token 4.2 us), many tokens the vector work of
 * turning levels into floats beside the products (16384 x 4096 by 128 bf16 tokens 45 us, 380 TFLOP/s).
 * fp32 has the most of it: by few tokens it bounds whole streams too (65536 x 4096 by one 34 us).
 */
#include <hip/hip_runtime.h>

#include "g53h.h"
#include "g53h_elem.h"
#include "g53h_runtime.h"

#define G53_W4_MAXE 1024
#define G53_W4_MAXC (1 << 24)          /* columns: 16 rows of levels or scales stay below 2^31 bytes */
#define G53_W4_MAXR (1 << 30)
#define G53_W4_NW 8                     /* waves of a workgroup, at most */
#define G53_W4_LDS_MAX (150 * 1024)
#define G53_W4_LDS (78 * 1024)          /* of its activations: two workgroups a CU */

struct G53W4Args {
    const uint8_t *w;                   /* levels [n][rows][cols / 2]                        */
    const void *s;                      /* scales [n][rows][groups], of type s_dt             */
    const uint8_t *z;                   /* zero points [n][rows][(groups + 1) / 2] or NULL: 8 */
    int rows, cols, group, groups, s_dt;
    int half;                           /* rows of the result (rows / 2 with SwiGLU)          */
    float limit;                        /* SwiGLU clamp, 0 without                            */
    int T;                              /* tokens, or sorted rows                             */
    const int *offsets;                 /* sorted rows: [n_experts + 1], else NULL            */
    const int *pair;                    /* sorted rows taken from tokens: pair / topk, or NULL */
    int n_experts, topk;
    long item0;                         /* first token tile of the launch                     */
    int tiles, items;                   /* row tiles, token tiles of the launch               */
    int kw_log;                         /* log2 of the parts that a workgroup's waves split the columns into */
    int glog;                           /* log2 of group / 32 where it is a power of two, else -1 */
    int seg;                            /* units of columns whose activations LDS holds       */
};

typedef unsigned int g53_v2w __attribute__((ext_vector_type(2)));

template <typename E> struct G53W4Type;   /* the 16-bit type of the products, planes per value */
template <> struct G53W4Type<float> { typedef g53_v8b V; static constexpr int P = 3; };
template <> struct G53W4Type<g53_bf16> { typedef g53_v8b V; static constexpr int P = 1; };
template <> struct G53W4Type<g53_f16> { typedef g53_v8h V; static constexpr int P = 1; };

__device__ __forceinline__ g53_v4f g53_mfma(g53_v8b a, g53_v8b b, g53_v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ g53_v4f g53_mfma(g53_v8h a, g53_v8h b, g53_v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

/* What takes a zero point z off levels, for g53_w4_levels: in each byte 128 - z (fp32), in each half -z as fp16; bf16: -z,
 * which takes it off the sum. */
template <typename E> __device__ __forceinline__ unsigned g53_w4_zero(unsigned z)
{
    if constexpr (__is_same(E, float)) return __builtin_amdgcn_perm(0u, 128u - z, 0u);
    if constexpr (__is_same(E, g53_bf16)) return __builtin_bit_cast(unsigned, -(float)z);
    return __builtin_amdgcn_perm(0u, __builtin_bit_cast(unsigned short, (g53_f16)(short)-(int)z), 0x01000100u);
}

/* Eight levels (nibbles 0..7 of d) in the order 0 2 1 3 4 6 5 7, less their zero point but for bf16. e4m3 codes 0 to 15,
 * those below the normal range and the first octave, are multiples of 2^-9, so a conversion takes two levels. */
template <typename E> __device__ __forceinline__ typename G53W4Type<E>::V g53_w4_levels(unsigned d, unsigned zero);
template <> __device__ __forceinline__ g53_v8b g53_w4_levels<float>(unsigned d, unsigned zero)
{
    /* bytes q + 128 - z, no carry between them, then q - z as signed bytes: even levels, odd levels */
    const unsigned even = ((d & 0x0f0f0f0fu) + zero) ^ 0x80808080u, odd = ((d >> 4 & 0x0f0f0f0fu) + zero) ^ 0x80808080u;
    g53_v4w o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned b = (i & 1 ? odd : even) >> 16 * (i >> 1);
        const float low = (float)(int)(int8_t)b, high = (float)(int)(int8_t)(b >> 8);
        o[i] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, high), __builtin_bit_cast(unsigned, low), 0x07060302u);
    }
    return __builtin_bit_cast(g53_v8b, o);
}
template <> __device__ __forceinline__ g53_v8b g53_w4_levels<g53_bf16>(unsigned d, unsigned)
{
    typedef g53_bf16 V2 __attribute__((ext_vector_type(2)));
    const unsigned even = d & 0x0f0f0f0fu, odd = d >> 4 & 0x0f0f0f0fu;
    const V2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, false);
    const V2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, false);
    const V2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, true);
    const V2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, true);
    return (g53_v8b){a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}
template <> __device__ __forceinline__ g53_v8h g53_w4_levels<g53_f16>(unsigned d, unsigned zero)
{
    typedef g53_f16 V2 __attribute__((ext_vector_type(2)));
    const unsigned even = d & 0x0f0f0f0fu, odd = d >> 4 & 0x0f0f0f0fu;
    const V2 z = __builtin_bit_cast(V2, zero);
    const V2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, false) + z;
    const V2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, false) + z;
    const V2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, true) + z;
    const V2 e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, true) + z;
    return (g53_v8h){a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

/* Eight activations in the levels' order, as P planes of the products' type. fp16: where one is not finite, the first pair
 * takes a NaN, and with it the row's results. (What is 0 times each, summed up: 0, or a NaN whose upper half is one of fp16.
 * fp32's second plane does it, infinity less itself, and bf16's sum of x.) */
template <typename V> __device__ __forceinline__ void g53_w4_x(V (&o)[1], const g53_v4w (&p)[1])
{
    const g53_v4w v = p[0];                                   /* 01 23 45 67 */
    unsigned none = 0u;
    if constexpr (__is_same(V, g53_v8h)) {
        typedef g53_f16 V2 __attribute__((ext_vector_type(2)));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned w = v[i];
            sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(V2, w), (V2){0.0f, 0.0f}, sum, false);
        }
        none = __builtin_bit_cast(unsigned, sum);
    }
    o[0] = __builtin_bit_cast(V, (g53_v4w){__builtin_amdgcn_perm(v[1], v[0], 0x05040100u) | none,
                                           __builtin_amdgcn_perm(v[1], v[0], 0x07060302u),
                                           __builtin_amdgcn_perm(v[3], v[2], 0x05040100u),
                                           __builtin_amdgcn_perm(v[3], v[2], 0x07060302u)});
}
__device__ __forceinline__ void g53_w4_x(g53_v8b (&o)[3], const g53_v4w (&p)[2])
{
    const g53_v4w a = p[0], b = p[1];
    unsigned v[8] = {a[0], a[2], a[1], a[3], b[0], b[2], b[1], b[3]};        /* 0 2 1 3 4 6 5 7 */
#pragma unroll
    for (int k = 0; k < 3; k++) {
        g53_v4w h;
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x07060302u);
        o[k] = __builtin_bit_cast(g53_v8b, h);
        if (k < 2)
#pragma unroll
            for (int i = 0; i < 8; i++)     /* what the upper half leaves: exact */
                v[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(float, v[i]) -
                                                        __builtin_bit_cast(float, v[i] & 0xffff0000u));
    }
}

/* Register s of the lanes' quarter q <-> register q of quarter s. */
__device__ __forceinline__ void g53_turn(unsigned (&d)[4])
{
    g53_v2w p;
    p = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
    d[0] = p[0]; d[2] = p[1];
    p = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
    d[1] = p[0]; d[3] = p[1];
    p = __builtin_amdgcn_permlane16_swap(d[0], d[1], false, false);
    d[0] = p[0]; d[1] = p[1];
    p = __builtin_amdgcn_permlane16_swap(d[2], d[3], false, false);
    d[2] = p[0]; d[3] = p[1];
}

/* The token tile `item` of the sorted rows: tiles of TT rows, expert by expert. False behind the last. */
__device__ __forceinline__ bool g53_w4_item(const int *__restrict__ offsets, int n_experts, long item, int TT,
                                            int &e, int &first, int &last)
{
    const int lane = threadIdx.x & 63, per = (n_experts + 63) / 64, e0 = lane * per;
    int n = 0, from = e0 < n_experts ? offsets[e0] : 0;
    for (int i = 0, at = from; i < per; i++)
        if (e0 + i < n_experts) {
            const int to = offsets[e0 + i + 1];
            n += (int)((unsigned)(to - at + TT - 1) / TT);
            at = to;
        }
    int incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
    }
    const unsigned long long in = __ballot((long)incl > item);
    if (!in) return false;
    const int l = __builtin_ctzll(in);
    int skip = (int)item - __builtin_amdgcn_readlane(incl - n, l);
    first = __builtin_amdgcn_readlane(from, l);
    for (e = l * per;; e++) {                 /* lane l's experts: one of them holds the tile */
        last = offsets[e + 1];
        const int tiles = (int)((unsigned)(last - first + TT - 1) / TT);
        if (skip < tiles) break;
        skip -= tiles;
        first = last;
    }
    first += skip * TT;
    last = last - first > TT ? first + TT : last;
    return true;
}

/* What a wave has asked for of 128 columns: levels of its row tiles as they lie, and, where they are not asked for by unit,
 * scales and zero points. */
template <int R, int X> struct G53W4Chunk {
    g53_v4w w[R];
    unsigned s[R], z[R];
    g53_v4w x[4][X];                    /* and of its activations, where LDS does not hold them: 8 columns a step */
};

/* n / d for 0 <= n, by a shift where d is a power of two (log >= 0). */
__device__ __forceinline__ int g53_quot(int n, int d, int log) { return log >= 0 ? n >> log : n / d; }

/* Every quarter's v to all lanes of its row: o[i] is quarter i's. */
__device__ __forceinline__ void g53_spread(unsigned (&o)[4], unsigned v)
{
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = v;
    g53_turn(o);
}
__device__ __forceinline__ void g53_spread(float (&o)[4], float v)
{
    unsigned u[4];
    g53_spread(u, __builtin_bit_cast(unsigned, v));
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = __builtin_bit_cast(float, u[i]);
}

/* One workgroup: up to 16 NT tokens (or sorted rows of one expert) by `out` (NW / KW) rows. Its waves are KW parts of the
 * columns, in units of UC x 128 taken in turn, by NW / KW groups of R row tiles. A unit's levels are asked for one unit
 * ahead. GS: groups are multiples of GS x 32 columns (4, 2 or 1). With SwiGLU the first R / 2 row tiles are gate rows,
 * the others the same up rows. Columns behind the last of a unit meet activations of zero. DIRECT (R = NT = 1): a wave
 * loads its activations a unit ahead into registers, from the caches, and LDS only adds up. */
template <typename E, int R, int NT, int UC, bool ROWS, bool LINES, bool DIRECT, int GS>
__global__ void __launch_bounds__(64 * G53_W4_NW, NT * G53W4Type<E>::P <= 3 ? 4 : 2)
k_w4(E *__restrict__ y, const E *__restrict__ x, const int *__restrict__ offsets, const int *__restrict__ pair, G53W4Args a)
{
    typedef typename G53W4Type<E>::V V;
    constexpr int P = G53W4Type<E>::P, PM = ROWS ? 1 : P, MT = 16 * NT, TT = ROWS ? MT / P : MT, LD = 16 * R + 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const bool sw = a.limit > 0.0f;
    const int out = sw ? 8 * R : 16 * R;                     /* result rows of a wave */
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), NW = blockDim.x >> 6;
    const int m = lane & 15, q = lane >> 4;
    const int KW = 1 << a.kw_log, kw = wv & (KW - 1), rw = wv >> a.kw_log, RW = NW >> a.kw_log;
    /* Workgroups go to the 8 dies in turn. Of one matrix, eight row tiles go side by side and a row tile's token tiles
     * after each other on one die, whose cache then holds the rows; of several, a token tile's row tiles follow each other. */
    const unsigned eight = 8u * a.items;
    const int tile = offsets ? blockIdx.x % a.tiles : blockIdx.x / eight * 8 + blockIdx.x % 8;
    if (tile >= a.tiles) return;
    const long item = a.item0 + (offsets ? blockIdx.x / a.tiles : blockIdx.x % eight / 8);
    int e = 0, first, last;
    if (offsets) {
        if (!g53_w4_item(offsets, a.n_experts, item, TT, e, first, last)) return;
        e = __builtin_amdgcn_readfirstlane(e);
        first = __builtin_amdgcn_readfirstlane(first);
        last = __builtin_amdgcn_readfirstlane(last);
    } else {
        first = (int)(item * TT);
        last = a.T - first < TT ? a.T : first + TT;
    }
    const int rows = last - first, x_rows = ROWS ? P * rows : rows, row0 = (tile * RW + rw) * out;
    /* where the row tiles begin; the lane's row in them, the last one for those behind the end */
    const uint8_t *wb[R], *sb[R], *zb[R];
    const int wrow = a.cols / 2, srow = a.groups * (a.s_dt == G53H_F32 ? 4 : 2), zrow = (a.groups + 1) / 2;
    int w_of[R][2], s_of[R], z_of[R];       /* the rows that the lane loads; the row m whose scales it takes */
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool up = sw && r >= R / 2;
        const int j = row0 + 16 * (up ? r - R / 2 : r), top = j < a.half ? j : a.half - 1;
        const int i = m < a.half - top ? m : a.half - top - 1;
        const long at = (long)e * a.rows + top + (up ? a.half : 0);
        wb[r] = a.w + at * wrow;
        sb[r] = (const uint8_t *)a.s + at * srow;
        zb[r] = a.z + at * zrow;
        const int end = a.half - top - 1;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int j8 = LINES ? (m & 7) + 8 * b : m;
            w_of[r][b] = (j8 < end ? j8 : end) * wrow;
        }
        s_of[r] = i * srow;
        z_of[r] = i * zrow;
    }
    g53_v4f acc[R][NT];
    const g53_v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < R; r++) acc[r][t] = zero;
    V ones;                             /* bf16: for the sums of x */
#pragma unroll
    for (int i = 0; i < 8; i++) ones[i] = 1.0f;
    const int units = (a.cols + 128 * UC - 1) / (128 * UC);

    /* scales and zero points of a group, as they lie, and as they enter */
    auto ask = [&](unsigned (&ks)[R], unsigned (&kz)[R], int g) {
        if (a.s_dt == G53H_F32)
#pragma unroll
            for (int r = 0; r < R; r++) ks[r] = *(const unsigned *)(sb[r] + (unsigned)(s_of[r] + g * 4));
        else
#pragma unroll
            for (int r = 0; r < R; r++) ks[r] = *(const uint16_t *)(sb[r] + (unsigned)(s_of[r] + g * 2));
        if (a.z)
#pragma unroll
            for (int r = 0; r < R; r++) kz[r] = zb[r][(unsigned)(z_of[r] + (g >> 1))];
    };
    /* a scale as it lies to fp32, without a branch: fp32 as it is, bf16 shifted, fp16 converted */
    const int s_shift = a.s_dt == G53H_BF16 ? 16 : 0;
    const unsigned s_f16 = a.s_dt == G53H_F16 ? ~0u : 0u, z_mask = a.z ? 15u : 0u, z_no = a.z ? 0u : 8u;
    auto scale = [&](unsigned v) {
        const float f16 = (float)__builtin_bit_cast(g53_f16, (uint16_t)v);
        return __builtin_bit_cast(float, (v << s_shift & ~s_f16) | (__builtin_bit_cast(unsigned, f16) & s_f16));
    };
    auto zero_of = [&](unsigned v, int g) { return g53_w4_zero<E>((v >> (4 * (g & 1)) & z_mask) | z_no); };
    /* the lane's group in chunk c: that of its quarter; in unit u: that of chunk q's half h (of NH halves) */
    constexpr int NH = GS == 4 ? 1 : 2;
    /* Scales are asked for by unit: by chunk they are as many requests to the vector cache as the levels (16384 x 4096 in
     * groups of 64 by one bf16 token 16.0 us against 12.2, by 5 fp16 tokens 16.6 against 12.8, 64 matrices of 2048 x 1024 by
     * 64 tokens 21.5 against 18.1; 4096 x 4096 by 64 fp32 tokens 30.6 either way). Not those of groups of 32, whose registers
     * would be too many. */
    constexpr bool UNIT = GS == 4 || (GS == 2 && UC > 1);
    auto group_of = [&](int c) {
        const int g = g53_quot(c * 4 + q, a.group / 32, a.glog);
        return g < a.groups ? g : a.groups - 1;
    };
    auto unit_group = [&](int u, int h) {
        const int g = g53_quot((u * UC + q) * 4 + 2 * h, a.group / 32, a.glog);
        return g < a.groups ? g : a.groups - 1;
    };
    constexpr int XW = sizeof(E) / 2;       /* 16-byte words of 8 activations */
    typedef G53W4Chunk<R, XW> Chunk;
    const E *xr = x;                        /* DIRECT: the lane's token */
    if (DIRECT) {
        const int i = first + (m < rows ? m : rows - 1), t = pair ? pair[i] / a.topk : i;
        xr = x + (long)t * a.cols + q * (GS == 4 ? 32 : 8);
    }
    /* Levels of a chunk, 16 rows x 64 bytes a load, or (LINES) of two: a load takes whole lines then, 8 rows x 128 bytes,
     * the first chunk's quarter q in lanes m < 8 of its rows and the second's in lanes m >= 8, until `pass` gives each lane
     * its row of both; such lines are not kept in the caches, where half lines wait for their other half. */
    constexpr int PAIR = LINES ? 2 : 1;
    auto load = [&](Chunk *k, int c) {
        const int w_at = c * 64 + (LINES ? (m >> 3) * 64 : 0) + q * 16;
        const int wo = w_at < wrow ? w_at : 0;      /* behind the end: not used */
#pragma unroll
        for (int b = 0; b < PAIR; b++)
#pragma unroll
            for (int r = 0; r < R; r++) {
                const g53_v4w *from = (const g53_v4w *)(wb[r] + (unsigned)(w_of[r][b] + wo));
                k[b].w[r] = LINES ? __builtin_nontemporal_load(from) : *from;
            }
        if (!UNIT)
#pragma unroll
            for (int b = 0; b < PAIR; b++) ask(k[b].s, k[b].z, group_of(c + b));
        if (DIRECT)
#pragma unroll
            for (int b = 0; b < PAIR; b++)
#pragma unroll
                for (int s = 0; s < 4; s++) {   /* columns behind the last: the row's first, made zero in `use` */
                    const int at = (c + b) * 128 + s * (GS == 4 ? 8 : 32);
                    const bool in = (GS == 4 ? (c + b) * 128 + q * 32 : at) < a.cols;
#pragma unroll
                    for (int j = 0; j < XW; j++) k[b].x[s][j] = ((const G53v4w_any *)(xr + (in ? at : 0)))[j].v;
                }
    };
    auto pass = [&](Chunk *k) {
        if (LINES)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) {       /* by 8 lanes of 16: rows 8..15 of the first, 0..7 of the second */
                    const int u = (int)k[0].w[r][i], v = (int)k[PAIR - 1].w[r][i];
                    k[0].w[r][i] = (unsigned)__builtin_amdgcn_update_dpp(u, v, 0x128, 0xf, 0xc, false);
                    k[PAIR - 1].w[r][i] = (unsigned)__builtin_amdgcn_update_dpp(v, u, 0x128, 0xf, 0x3, false);
                }
    };
    const int ld = a.seg * (256 * UC) + 16; /* bytes of a plane's row in LDS: odd sixteens, so rows start in other banks */
    int xat[NT];                            /* the lane's token in LDS; tokens behind the last repeat it */
#pragma unroll
    for (int t = 0; t < NT; t++) xat[t] = (16 * t + m < x_rows ? 16 * t + m : x_rows - 1) * ld + q * (GS == 4 ? 64 : 16);
    const int plane = rows * ld;
    /* sc4, zr4: of the chunk's halves, where UNIT. Step s takes the columns of register s: 8 from each quarter's 32 where
     * the chunk lies in one group, else turned to 32 in a row. */
    auto use = [&](const Chunk &k, int c, int c_lds, const float (&sc4)[R][NH], const unsigned (&zr4)[R][NH]) {
        unsigned d[R][4], zr[R][4];
        float sc[R][4];
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
            for (int i = 0; i < 4; i++) d[r][i] = k.w[r][i];
            if (GS < 4) g53_turn(d[r]);
            if (UNIT) {
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    sc[r][GS * (h + 1) - 1] = sc4[r][h];
#pragma unroll
                    for (int i = 0; i < GS; i++) zr[r][GS * h + i] = zr4[r][h];
                }
            } else {
                g53_spread(sc[r], scale(k.s[r]));
                g53_spread(zr[r], zero_of(k.z[r], group_of(c)));
            }
        }
        /* the upper planes of fp32 apart from the lower ones, whose roundings are 2^-8 of theirs then */
        constexpr int DP = PM == 3 ? 2 : 1;
        constexpr bool SUM = __is_same(E, g53_bf16);    /* zero points come off the sums, with x's */
        g53_v4f D[R][NT][DP], X[NT];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            V b[NT][PM];
            if (DIRECT) {
                V o[P];
                g53_v4w v[XW];
                const bool in = c * 128 + (GS == 4 ? q : s) * 32 < a.cols;
#pragma unroll
                for (int j = 0; j < XW; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) v[j][i] = in ? k.x[s][j][i] : 0u;
                g53_w4_x(o, v);
#pragma unroll
                for (int p = 0; p < PM; p++) b[0][p] = o[p];
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int p = 0; p < PM; p++) {
                    if (!DIRECT) b[t][p] = *(const V *)(lds + p * plane + xat[t] + c_lds * 256 + s * (GS == 4 ? 16 : 64));
                    if (SUM) X[t] = g53_mfma(b[t][p], ones, s % GS == 0 ? zero : X[t]);
                }
#pragma unroll
            for (int r = 0; r < R; r++) {
                const V lv = g53_w4_levels<E>(d[r][s], zr[r][s]);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int p = 0; p < PM; p++) {
                        g53_v4f &to = D[r][t][p ? DP - 1 : 0];
                        to = g53_mfma(b[t][p], lv, s % GS == 0 && p < 2 ? zero : to);
                    }
            }
            if (NT * PM > 2) __builtin_amdgcn_sched_barrier(0);     /* one step's activations in registers at a time */
            if (s % GS == GS - 1)       /* a group, or what the chunk has of it */
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int t = 0; t < NT; t++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            float v = D[r][t][0][i];
                            if (SUM) v = __builtin_fmaf(__builtin_bit_cast(float, zr[r][s]), X[t][i], v);
                            if (DP == 2) v += D[r][t][DP - 1][i];
                            acc[r][t][i] = __builtin_fmaf(sc[r][s], v, acc[r][t][i]);
                        }
                        asm volatile("" : "+v"(acc[r][t]));      /* added here, not behind the next branch with D kept */
                    }
        }
        __builtin_amdgcn_sched_barrier(0);      /* no work on the next chunk, which may not be there yet, before this is done */
    };
    Chunk ring[UC];
    /* a unit's scales, where UNIT: quarter i holds those of chunk i */
    unsigned us[NH][R], uz[NH][R];
    auto ask_unit = [&](int u) {
        if (UNIT)
#pragma unroll
            for (int h = 0; h < NH; h++) ask(us[h], uz[h], unit_group(u, h));
    };
    auto unit_scales = [&](int u, float (&sc)[NH][R][4], unsigned (&zr)[NH][R][4]) {
        if (UNIT)
#pragma unroll
            for (int h = 0; h < NH; h++) {
                const int g = unit_group(u, h);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    g53_spread(sc[h][r], scale(us[h][r]));
                    g53_spread(zr[h][r], zero_of(uz[h][r], g));
                }
            }
    };
    /* A segment's activations into LDS as planes in the levels' order, in pieces of 512 columns of a row, a wave's load;
     * a wave asks for NP at a time. */
    constexpr int NP = (P == 3 && R == 2) || NT > 1 ? 2 : 4;
    typedef g53_v4w Piece[NP][sizeof(E) / 2];
    auto segment = [&](int seg0) { return units - seg0 < a.seg ? units - seg0 : a.seg; };
    auto pieces_of = [&](int here) { return rows * ((here * (16 * UC) + 63) / 64); };
    auto fetch = [&](Piece &v, int seg0, int p0) {
        const int k0 = seg0 * (128 * UC), across = pieces_of(segment(seg0)) / rows;
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int piece = p0 + k * NW, i = piece / across, at = k0 + ((piece - i * across) * 64 + lane) * 8;
            const bool there = i < rows && at < a.cols;
            int p = i < rows ? first + i : first;
            if (pair) p = pair[p] / a.topk;
#pragma unroll
            for (int j = 0; j < (int)sizeof(E) / 2; j++) {
                v[k][j] = (g53_v4w){0, 0, 0, 0};
                if (there) v[k][j] = ((const G53v4w_any *)(x + (long)p * a.cols + at))[j].v;
            }
        }
    };
    auto put = [&](Piece &v, int seg0, int p0) {
        const int here = segment(seg0), across = pieces_of(here) / rows;
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int piece = p0 + k * NW, i = piece / across, c8 = (piece - i * across) * 64 + lane;
            if (i < rows && c8 < here * (16 * UC)) {
                V b[P];
                g53_w4_x(b, v[k]);
#pragma unroll
                for (int j = 0; j < P; j++) *(V *)(lds + j * plane + i * ld + c8 * 16) = b[j];
            }
        }
    };
    {   /* the first levels: behind the first activations, which LDS has to hold before */
        Piece v;
        if (!DIRECT) fetch(v, 0, wv);
        __builtin_amdgcn_sched_barrier(0);
        ask_unit(kw);
#pragma unroll
        for (int j = 0; j < UC; j += PAIR) load(ring + j, kw * UC + j);
        __builtin_amdgcn_sched_barrier(0);
        if (!DIRECT) put(v, 0, wv);
    }
    for (int seg0 = 0; seg0 < units; seg0 += a.seg) {
        const int here = segment(seg0), pieces = pieces_of(here);
        if (!DIRECT) {
            if (seg0) __syncthreads();
            for (int p0 = seg0 ? wv : wv + NP * NW; p0 < pieces; p0 += NP * NW) {
                Piece v;
                fetch(v, seg0, p0);
                put(v, seg0, p0);
            }
            __syncthreads();
        }
        /* every unit asks for the wave's next one, but for the last of all; segments but the last are whole turns */
        const bool ends = seg0 + here == units;
        const int until = ends ? here - KW : here;
        int i = kw;
        float sc[NH][R][4], sj[R][NH];
        unsigned zr[NH][R][4], zj[R][NH];
        for (; i < until; i += KW) {
            unit_scales(seg0 + i, sc, zr);
            ask_unit(seg0 + i + KW);
#pragma unroll
            for (int j = 0; j < UC; j++) {
                if (j % PAIR == 0) pass(ring + j);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int h = 0; h < NH; h++) { sj[r][h] = sc[h][r][j]; zj[r][h] = zr[h][r][j]; }
                use(ring[j], (seg0 + i) * UC + j, i * UC + j, sj, zj);
                if (j % PAIR == PAIR - 1) load(ring + j - (PAIR - 1), (seg0 + i + KW) * UC + j - (PAIR - 1));
            }
        }
        if (ends && i < here) {
            unit_scales(seg0 + i, sc, zr);
#pragma unroll
            for (int j = 0; j < UC; j++) {
                if (j % PAIR == 0) pass(ring + j);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int h = 0; h < NH; h++) { sj[r][h] = sc[h][r][j]; zj[r][h] = zr[h][r][j]; }
                use(ring[j], (seg0 + i) * UC + j, i * UC + j, sj, zj);
            }
        }
    }
    __syncthreads();
    float *red = (float *)lds;              /* [NW][MT][LD] */
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) red[(wv * MT + 16 * t + 4 * q + i) * LD + 16 * r + m] = acc[r][t][i];
    __syncthreads();
    /* out and RW are powers of two */
    const int out_log = __builtin_ctz(out), outs_log = out_log + __builtin_ctz(RW), base = tile << outs_log;
    for (int i = tid; i < rows << outs_log; i += 64 * NW) {
        const int t = i >> outs_log, o = i & ((1 << outs_log) - 1), w = o >> out_log, r = o & (out - 1);
        float v = 0.0f, u = 0.0f;
        for (int k = 0; k < KW; k++)
#pragma unroll
            for (int p = 0; p < (ROWS ? P : 1); p++) {
                const float *from = red + ((w * KW + k) * MT + p * rows + t) * LD + r;
                v += from[0];
                if (sw) u += from[out];
            }
        if (sw) {
            v = v > a.limit ? a.limit : v;
            u = u > a.limit ? a.limit : (u < -a.limit ? -a.limit : u);
            v = v / (1.0f + expf(-v)) * u;
        }
        if (base + o < a.half) y[(long)(first + t) * a.half + base + o] = (E)v;
    }
}

template <typename E, int R, int NT, int UC, bool ROWS, bool LINES, bool DIRECT, int GS>
static int start(dim3 grid, int waves, size_t lds, void *y, const void *x, const G53W4Args &a)
{
    static int allowed = 0;
    if (!allowed) {
        G53_TRY(hipFuncSetAttribute((const void *)k_w4<E, R, NT, UC, ROWS, LINES, DIRECT, GS>,
                                    hipFuncAttributeMaxDynamicSharedMemorySize, G53_W4_LDS_MAX));
        allowed = 1;
    }
    hipLaunchKernelGGL((k_w4<E, R, NT, UC, ROWS, LINES, DIRECT, GS>), grid, dim3(64 * waves), lds, g53h_stream(), (E *)y,
                       (const E *)x, a.offsets, a.pair, a);
    G53_LAUNCHED("k_w4");
    return 0;
}

/* busy: token tiles that are expected to hold rows, mean: rows of an expert. */
template <typename E, int R, int NT, int UC, bool ROWS, bool LINES = false, bool DIRECT = false>
static int launch(void *y, const void *x, G53W4Args &a, long items, long busy, long mean)
{
    constexpr int P = G53W4Type<E>::P, TT = ROWS ? 16 * NT / P : 16 * NT;
    const bool sw = a.limit > 0.0f;
    const int out = sw ? 8 * R : 16 * R, units = (a.cols + 128 * UC - 1) / (128 * UC), rows = a.T < TT ? a.T : TT;
    /* A workgroup's eight waves are rw groups of rows by 2^k parts of the columns. A workgroup takes the time that its
     * activations need on their way to LDS, as of 5 rows each, and its rows', and the CUs take workgroups in rounds: 8192 x
     * 4096 by 64 bf16 tokens 256 workgroups 18.8 us, 512 20.4, 128 28.5; 6000 x 4096 by 16: 188 11.0, 375 16.6; by 5 fp32
     * tokens 8192 x 4096: 256 9.9, 512 15.6. An expert's rows count as `mean`, all experts' alike, since the host does not know
     * them: uneven ones can do better by other parts (512 rows of each of 16 experts by 64 tokens 10.8, by twice the rows a
     * workgroup 9.0), and so can some single matrices (24576 x 2048 gate/up by one 11.9, by a quarter 10.8). DIRECT has no
     * activations in LDS to share: the fewest rows that leave two workgroups a CU. */
    int k = 0, rw = units < 4 ? G53_W4_NW / 2 : G53_W4_NW;
    const int each = mean < rows ? (int)mean : rows;
    long least = 0;
    for (int i = 0, r = rw;; r /= 2) {
        const long wgs = busy * ((a.half + out * r - 1) / (out * r)), slots = g53h_num_cus() * (G53_W4_NW / (r << i));
        const long cost = (wgs + slots - 1) / slots * (G53_W4_NW / (r << i)) * (5 * each + out * r);
        if (DIRECT || !least || cost < least) {
            least = cost;
            rw = r;
            k = i;
        }
        if (r == 1 || (DIRECT && wgs >= 2 * g53h_num_cus())) break;
        if ((2 << i) <= units && (DIRECT || rows * P * ((2 << i) * 256 * UC + 16) <= G53_W4_LDS_MAX)) i++;
    }
    if (DIRECT && (rw > 1 || (busy * ((a.half + out - 1) / out) << k) > 8 * g53h_num_cus())) return 1;
    const int waves = rw << k, outs = out * rw;
    a.kw_log = k;
    a.tiles = (a.half + outs - 1) / outs;
    int seg = (G53_W4_LDS / (rows * P) - 16) / (256 * UC) >> k << k;    /* units of x in LDS: whole turns */
    if (seg < 1 << k) seg = 1 << k;
    if (seg > units || DIRECT) seg = units;
    a.seg = seg;
    size_t lds = DIRECT ? 0 : (size_t)rows * P * (seg * 256 * UC + 16), red = (size_t)waves * 16 * NT * (16 * R + 4) * 4;
    if (lds < red) lds = red;
    /* threads of a launch, 64 a wave, fit 32 bits: waves are as many as groups of rows (rw) where rows pass 2^29, so 2^30
     * rows are 2^31 threads at least, of 32 rows a wave */
    const long wide = a.offsets ? a.tiles : (a.tiles + 7) / 8 * 8l, most = (1l << 31) / (64 * waves) / wide;
    if (most < 1) return g53h_fail("4-bit product: %d rows in workgroups of %d rows and %d waves", a.rows, outs, waves);
    for (long i = 0; i < items; i += most) {
        a.item0 = i;
        a.items = (int)(items - i < most ? items - i : most);
        const dim3 grid((unsigned)(a.items * wide));
        const int rc = a.group % 128 == 0 ? start<E, R, NT, UC, ROWS, LINES, DIRECT, 4>(grid, waves, lds, y, x, a)
                       : a.group % 64 == 0 ? start<E, R, NT, UC, ROWS, LINES, DIRECT, 2>(grid, waves, lds, y, x, a)
                                           : start<E, R, NT, UC, ROWS, LINES, DIRECT, 1>(grid, waves, lds, y, x, a);
        if (rc) return rc;
    }
    return 0;
}

/* Row tiles of a wave: two, so that activations read from LDS meet twice the levels, or one where two leave less than
 * 16 waves a CU (4096 x 2048 by one token in bf16, both with LDS: 5.6 us against 8.0). Token tiles of 16, or of 32 for more
 * tokens where they leave 32 waves a CU, which then turn levels into floats half as often (16384 x 4096 by 128 tokens in
 * bf16 45.4 us against 48.2, in fp16 44.6 against 50.0; 8192 x 4096 by 64, of fewer waves, 21.7 against 18.5; in fp32, whose
 * waves take twice the registers then, 8192 x 4096 by 128 in groups of 64 54 against 66, but 16384 x 4096 by 128 90 against
 * 81 and 64 gate/up experts of 2048 x 2048 by 256 tokens 141 against 100).
 * For fp32, whose products are three, up to 5 tokens put their planes side by side as 15 rows of a tile, and
 * the products are as many as bf16's (16384 x 4096 by one token: 11.4 us against 18.0). Long rows of a matrix that one
 * token tile meets are loaded in whole lines (65536 x 4096 by 5 fp16 tokens: 30.0 us against 33.3; eight gate/up matrices of
 * 4096 x 4096 by one token 17.0 against 18.5); short rows, or rows that further tiles read again, in half lines (64 matrices
 * of 2048 x 1024 by 64 tokens 17.9 against 18.4, 8192 x 4096 by 64 18.5 against 18.9).
 * Small matrices, of at most 8 waves a CU that share no activations, load them without LDS, which takes a trip to memory
 * and a barrier out of a call that is little else: 4096 x 2048 by one token in bf16 4.2 us against 5.6, 1001 x 2080 by 24 in
 * fp32 7.2 against 10.2, one expert's 1024 x 1024 by one 4.0 against 5.0; of more waves the caches' rate bounds them
 * (4096 x 4096 by 8 tokens in bf16 6.4 either way, 6000 x 4096 10.2 against 8.0). Up to 5 fp32 tokens do so where a wave has
 * at most two chunks (256 x 512 by one 3.5 against 4.4; 4096 x 4096 by one 8.6 against 6.5). */
template <typename E> static int by_tokens(void *y, const void *x, G53W4Args &a)
{
    constexpr bool F32 = sizeof(E) == 4;
    const long ex = a.offsets ? (a.n_experts < a.T ? a.n_experts : a.T) : 1, mean = (a.T + ex - 1) / ex;
    const long units = (a.cols + 511) / 512;
    const long waves = (a.rows + 31) / 32 * ex * ((mean + 15) / 16) * (units < G53_W4_NW ? units : G53_W4_NW);
    const bool few = waves <= 16 * g53h_num_cus() && !(a.limit > 0.0f);
    const long waves32 = (a.rows + 31) / 32 * ex * ((mean + 31) / 32) * (units < G53_W4_NW ? units : G53_W4_NW);
    const bool many = waves32 >= 32 * g53h_num_cus();
    const int TT = F32 && mean <= 5 ? 5 : (mean > 16 && many ? 32 : 16);
    auto items_of = [&](int tt) { return a.offsets ? a.T / tt + ex : (a.T - 1) / tt + 1l; };
    auto busy_of = [&](int tt) { return ex * ((mean + tt - 1) / tt); };
    const long items = items_of(TT), busy = busy_of(TT);
    if (TT == 32) return launch<E, 2, 2, 2, false>(y, x, a, items, busy, mean);
    if (few && (TT == 16 || a.cols <= 2048)) {
        const int rc = launch<E, 1, 1, F32 ? 1 : 2, false, false, true>(y, x, a, items_of(16), busy_of(16), mean);
        if (rc <= 0) return rc;
    }
    if constexpr (F32)
        if (TT == 16)
            return few ? launch<E, 1, 1, 1, false>(y, x, a, items, busy, mean) : launch<E, 2, 1, 2, false>(y, x, a, items, busy, mean);
    if (few) return launch<E, 1, 1, 4, F32>(y, x, a, items, busy, mean);
    if (mean <= TT && units >= 4) return launch<E, 2, 1, 4, F32, true>(y, x, a, items, busy, mean);
    return launch<E, 2, 1, 4, F32>(y, x, a, items, busy, mean);
}

static int product(void *y, const void *x, int dt, G53W4Args &a)
{
    if (g53h_ready()) return -1;
    int rc;
    G53_BY_TYPE(dt, rc = by_tokens<E>(y, x, a));
    return rc;
}

static int w4_bad(const char *who, const G53hW4 *m, int dt, float limit, G53W4Args &a)
{
    if (!m || !m->w || !m->s) return g53h_fail("%s: unbound matrix", who);
    if (m->rows < 1 || m->rows > G53_W4_MAXR || m->cols < 32 || m->cols > G53_W4_MAXC || m->cols % 32 || m->group < 32 ||
        m->group % 32 || !g53_elem_bytes(m->s_dt))
        return g53h_fail("%s: %d x %d levels in groups of %d, scale type %d (columns and group multiples of 32, at most 2^24 "
                         "columns of 2^30 rows)", who, m->rows, m->cols, m->group, m->s_dt);
    if (((uintptr_t)m->w & 15) || ((uintptr_t)m->s & (g53_elem_bytes(m->s_dt) - 1)))
        return g53h_fail("%s: levels must start at a multiple of 16 bytes, scales of their type", who);
    if (!g53_elem_bytes(dt)) return g53h_fail("%s: element type %d", who, dt);
    if (!(limit >= 0.0f) || limit > 3.0e38f) return g53h_fail("%s: SwiGLU limit %g", who, limit);
    if (limit > 0.0f && m->rows % 2) return g53h_fail("%s: SwiGLU of %d rows", who, m->rows);
    a.w = m->w;
    a.s = m->s;
    a.z = m->z;
    a.rows = m->rows;
    a.cols = m->cols;
    a.group = m->group < m->cols ? m->group : m->cols;
    a.groups = (m->cols - 1) / a.group + 1;
    a.s_dt = m->s_dt;
    a.glog = (a.group & (a.group - 1)) ? -1 : __builtin_ctz(a.group) - 5;
    a.limit = limit;
    a.half = limit > 0.0f ? m->rows / 2 : m->rows;
    a.offsets = a.pair = nullptr;
    a.n_experts = a.topk = 1;
    a.item0 = 0;
    a.tiles = a.items = a.kw_log = a.seg = 0;
    return 0;
}

extern "C" int g53h_mm_w4(void *y, const void *x, int dt, int T, const G53hW4 *m, float swiglu_limit)
{
    G53W4Args a;
    if (w4_bad("g53h_mm_w4", m, dt, swiglu_limit, a)) return -1;
    if (T < 0) return g53h_fail("g53h_mm_w4: %d tokens", T);
    if (!T) return 0;
    if (!y || !x) return g53h_fail("g53h_mm_w4: no tokens");
    a.T = T;
    return product(y, x, dt, a);
}

extern "C" int g53h_sorted_mm_w4(void *ys, const void *x, int dt, int gather, const G53hSort *p, const G53hW4 *m,
                                 float swiglu_limit)
{
    G53W4Args a;
    if (w4_bad("g53h_sorted_mm_w4", m, dt, swiglu_limit, a)) return -1;
    if (!p || p->T < 0 || p->topk < 1 || p->topk > 64 || p->n_experts < 1 || p->n_experts > G53_W4_MAXE ||
        (long)p->T * p->topk > 0x7fffffffl || !p->offsets || (p->T && !p->pair))
        return g53h_fail("g53h_sorted_mm_w4: no plan of g53h_sort_tokens");
    if (!p->T) return 0;
    if (!ys || !x) return g53h_fail("g53h_sorted_mm_w4: no rows");
    a.T = p->T * p->topk;
    a.offsets = p->offsets;
    a.pair = gather ? p->pair : nullptr;
    a.n_experts = p->n_experts;
    a.topk = p->topk;
    return product(ys, x, dt, a);
}
