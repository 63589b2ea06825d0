/* g53h_w4.hip - products of a few tokens with matrices of 4-bit levels and group scales, of one
 * matrix (g53h_mm_w4) or of the matrix of each sorted row's expert (g53h_sorted_mm_w4):
 *
 *     y[t][r] = sum over groups g of  s[r][g] * sum over c in g of (q[r][c] - z[r][g]) x[t][c]
 *
 * Levels go to the matrix cores as they are, without a multiplication: level q becomes the 16-bit
 * float 16 + q (its four bits are the top bits of the mantissa of 2^4), one shift and one and-or per
 * two levels, exact in bf16 and fp16. What was added comes off per group: with X = the group's sum of
 * x (one product with a matrix of ones, shared by all row tiles), the group adds s (D - (16 + z) X).
 * Products are exact in fp32 and summed in fp32; fp32 activations enter as three bf16 planes whose sum
 * is the value exactly (8 + 8 + 8 mantissa bits, by truncation).
 *
 * A wave owns R tiles of 16 rows and NT tiles of 16 tokens over a part of the columns and steps by 128
 * columns: one 16-byte load per lane and row tile (16 rows x 64 bytes), turned so that each of the
 * four products of 32 columns covers consecutive columns (v_permlane32_swap and v_permlane16_swap
 * exchange the lanes' quarters with the four registers), so groups of any multiple of 32 end between
 * products. The NW waves of a workgroup split the columns and add up through LDS.
 */
#include <hip/hip_runtime.h>

#include "g53h.h"
#include "g53h_elem.h"
#include "g53h_runtime.h"

#define G53_W4_MAXE 1024

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
    int tiles;                          /* row tiles                                          */
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

/* Eight levels (nibbles 0..7 of d) as 16 + level, in the order 0 4 1 5 2 6 3 7. */
template <typename V> __device__ __forceinline__ V g53_w4_levels(unsigned d);
template <> __device__ __forceinline__ g53_v8b g53_w4_levels<g53_v8b>(unsigned d)
{
    const unsigned m = 0x00780078u, o = 0x41804180u;          /* bf16 16.0, mantissa bits 6..3 */
    return __builtin_bit_cast(g53_v8b, (g53_v4w){((d << 3) & m) | o, ((d >> 1) & m) | o, ((d >> 5) & m) | o,
                                                 ((d >> 9) & m) | o});
}
template <> __device__ __forceinline__ g53_v8h g53_w4_levels<g53_v8h>(unsigned d)
{
    const unsigned m = 0x03c003c0u, o = 0x4c004c00u;          /* fp16 16.0, mantissa bits 9..6 */
    return __builtin_bit_cast(g53_v8h, (g53_v4w){((d << 6) & m) | o, ((d << 2) & m) | o, ((d >> 2) & m) | o,
                                                 ((d >> 6) & m) | o});
}

/* Eight activations from p in the levels' order, as P planes of the products' type. */
template <typename V> __device__ __forceinline__ void g53_w4_x16(V (&o)[1], const void *p)
{
    const g53_v4w v = ((const G53v4w_any *)p)->v;              /* 01 23 45 67 */
    o[0] = __builtin_bit_cast(V, (g53_v4w){__builtin_amdgcn_perm(v[2], v[0], 0x05040100u),
                                           __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                                           __builtin_amdgcn_perm(v[3], v[1], 0x05040100u),
                                           __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)});
}
__device__ __forceinline__ void g53_w4_x(g53_v8b (&o)[1], const g53_bf16 *p) { g53_w4_x16(o, p); }
__device__ __forceinline__ void g53_w4_x(g53_v8h (&o)[1], const g53_f16 *p) { g53_w4_x16(o, p); }
__device__ __forceinline__ void g53_w4_x(g53_v8b (&o)[3], const float *p)
{
    const g53_v4w a = ((const G53v4w_any *)p)[0].v, b = ((const G53v4w_any *)p)[1].v;
    unsigned v[8];
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = a[i]; v[2 * i + 1] = b[i]; }   /* 0 4 1 5 2 6 3 7 */
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

__device__ __forceinline__ float g53_w4_scale(const G53W4Args &a, long i)
{
    if (a.s_dt == G53H_F32) return ((const float *)a.s)[i];
    if (a.s_dt == G53H_BF16) return (float)((const g53_bf16 *)a.s)[i];
    return (float)((const g53_f16 *)a.s)[i];
}

/* The token tile `item` of the sorted rows: tiles of TT rows, expert by expert. False behind the last. */
__device__ __forceinline__ bool g53_w4_item(const G53W4Args &a, long item, int TT, int &e, int &first, int &last)
{
    const int lane = threadIdx.x & 63, per = (a.n_experts + 63) / 64, e0 = lane * per;
    int n = 0;
    for (int i = 0; i < per; i++)
        if (e0 + i < a.n_experts) n += (a.offsets[e0 + i + 1] - a.offsets[e0 + i] + TT - 1) / TT;
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
    for (e = l * per;; e++) {                 /* lane l's experts: one of them holds the tile */
        first = a.offsets[e];
        last = a.offsets[e + 1];
        const int tiles = (last - first + TT - 1) / TT;
        if (skip < tiles) break;
        skip -= tiles;
    }
    first += skip * TT;
    last = first + TT < last ? first + TT : last;
    return true;
}

/* SW: SwiGLU; the first R / 2 row tiles are gate rows, the others the same up rows. */
template <typename E, int R, int NT, int NW, bool SW>
__global__ void __launch_bounds__(64 * NW) k_w4(E *__restrict__ y, const E *__restrict__ x, G53W4Args a)
{
    typedef typename G53W4Type<E>::V V;
    constexpr int P = G53W4Type<E>::P, TT = 16 * NT, LD = 16 * R + 4;
    __shared__ float red[NW][TT][LD];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, q = lane >> 4;
    const long item = a.item0 + blockIdx.x / a.tiles;
    const int tile = blockIdx.x % a.tiles;
    int e = 0, first, last;
    if (a.offsets) {
        if (!g53_w4_item(a, item, TT, e, first, last)) return;
        e = __builtin_amdgcn_readfirstlane(e);
    } else {
        first = (int)(item * TT);
        last = a.T - first < TT ? a.T : first + TT;
    }
    constexpr int OUT = SW ? 8 * R : 16 * R;                 /* result rows of a workgroup */
    const int row0 = tile * OUT;
    /* row tile r starts at this row of the matrix */
    auto tile_row = [&](int r) { return SW ? (r < R / 2 ? row0 + 16 * r : a.half + row0 + 16 * (r - R / 2)) : row0 + 16 * r; };
    auto tile_end = [&](int r) { return SW && r < R / 2 ? a.half : a.rows; };
    const long wrow = a.cols / 2, mat = (long)e * a.rows, zrow = (a.groups + 1) / 2;
    const uint8_t *wp[R];
    long srow[R][4];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int end = tile_end(r) - 1;
        const int i = tile_row(r) + m;
        wp[r] = a.w + (mat + (i < end ? i : end)) * wrow + q * 16;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int j = tile_row(r) + 4 * q + k;
            srow[r][k] = mat + (j < end ? j : end);
        }
    }
    const E *xp[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        int p = first + 16 * t + m;
        p = p < last ? p : last - 1;                          /* columns behind the last repeat it and are not written */
        if (a.pair) p = a.pair[p] / a.topk;
        xp[t] = x + (long)p * a.cols + q * 8;
    }
    g53_v4f acc[R][NT], D[R][NT], X[NT];
    const g53_v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; t++) {
        X[t] = zero;
#pragma unroll
        for (int r = 0; r < R; r++) { acc[r][t] = zero; D[r][t] = zero; }
    }
    V ones;
#pragma unroll
    for (int i = 0; i < 8; i++) ones[i] = 1.0f;
    const int chunks = (a.cols + 127) / 128, per = (chunks + NW - 1) / NW;
    const int c0 = wv * per, c1 = c0 + per < chunks ? c0 + per : chunks;
    int g = c0 * 128 / a.group, left = (g + 1) * a.group - c0 * 128;      /* the group, and its columns to come */
    for (int c = c0; c < c1; c++) {
        unsigned d[R][4];
        const int steps = a.cols - c * 128 >= 128 ? 4 : (a.cols - c * 128) / 32;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const g53_v4w v = q < steps ? ((const G53v4w_any *)(wp[r] + c * 64))->v : (g53_v4w){0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; i++) d[r][i] = v[i];
            g53_turn(d[r]);
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            if (s < steps) {
                V b[NT][P];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    g53_w4_x(b[t], xp[t] + c * 128 + s * 32);
#pragma unroll
                    for (int k = 0; k < P; k++) X[t] = g53_mfma(ones, b[t][k], X[t]);
                }
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const V lv = g53_w4_levels<V>(d[r][s]);
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int k = 0; k < P; k++) D[r][t] = g53_mfma(lv, b[t][k], D[r][t]);
                }
                left -= 32;
                if (left == 0 || (c == c1 - 1 && s == steps - 1)) {     /* the group, or the wave's part, ends */
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float sc = g53_w4_scale(a, srow[r][i] * a.groups + g);
                            const float nz = a.z ? -16.0f - (float)((a.z[srow[r][i] * zrow + (g >> 1)] >> (4 * (g & 1))) & 15)
                                                 : -24.0f;
#pragma unroll
                            for (int t = 0; t < NT; t++)
                                acc[r][t][i] = __builtin_fmaf(sc, __builtin_fmaf(nz, X[t][i], D[r][t][i]), acc[r][t][i]);
                        }
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        X[t] = zero;
#pragma unroll
                        for (int r = 0; r < R; r++) D[r][t] = zero;
                    }
                    left = a.group;
                    g++;
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < NT; t++) *(g53_v4f *)&red[wv][16 * t + m][16 * r + 4 * q] = acc[r][t];
    __syncthreads();
    for (int i = tid; i < TT * OUT; i += 64 * NW) {
        const int t = i / OUT, r = i % OUT;
        float v = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            v += red[w][t][r];
            if (SW) u += red[w][t][OUT + r];
        }
        if (SW) {
            v = v > a.limit ? a.limit : v;
            u = u > a.limit ? a.limit : (u < -a.limit ? -a.limit : u);
            v = v / (1.0f + expf(-v)) * u;
        }
        if (first + t < last && row0 + r < a.half) y[(long)(first + t) * a.half + row0 + r] = (E)v;
    }
}

template <typename E, int R, int NT, int NW> static int launch(void *y, const void *x, G53W4Args &a, long items)
{
    const bool sw = a.limit > 0.0f;
    const int out = sw ? 8 * R : 16 * R;
    a.tiles = (a.half + out - 1) / out;
    const long most = (1l << 31) / (64 * NW) / a.tiles;      /* token tiles of one launch: threads fit 32 bits */
    if (most < 1) return g53h_fail("g53h_mm_w4: %d rows", a.rows);
    for (long i = 0; i < items; i += most) {
        a.item0 = i;
        const dim3 grid((unsigned)((items - i < most ? items - i : most) * a.tiles)), block(64 * NW);
        if (sw) hipLaunchKernelGGL((k_w4<E, R, NT, NW, true>), grid, block, 0, g53h_stream(), (E *)y, (const E *)x, a);
        else hipLaunchKernelGGL((k_w4<E, R, NT, NW, false>), grid, block, 0, g53h_stream(), (E *)y, (const E *)x, a);
        G53_LAUNCHED("k_w4");
    }
    return 0;
}

/* Tokens, or sorted rows, of the busiest matrix decide the tile. */
static int product(void *y, const void *x, int dt, G53W4Args &a)
{
    constexpr int NT = 1;
    const long tiles = ((long)a.T + 16 * NT - 1) / (16 * NT);
    const long items = a.offsets ? tiles + (a.n_experts < a.T ? a.n_experts : a.T) : tiles;
    if (g53h_ready()) return -1;
    int rc;
    G53_BY_TYPE(dt, rc = (launch<E, 2, NT, 8>(y, x, a, items)));
    return rc;
}

static int w4_bad(const char *who, const G53hW4 *m, int dt, float limit, G53W4Args &a)
{
    if (!m || !m->w || !m->s) return g53h_fail("%s: unbound matrix", who);
    if (m->rows < 1 || m->cols < 32 || m->cols % 32 || m->group < 32 || m->group % 32 || !g53_elem_bytes(m->s_dt))
        return g53h_fail("%s: %d x %d levels in groups of %d, scale type %d (columns and group multiples of 32)", who, m->rows,
                         m->cols, m->group, m->s_dt);
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
    a.limit = limit;
    a.half = limit > 0.0f ? m->rows / 2 : m->rows;
    a.offsets = a.pair = nullptr;
    a.n_experts = a.topk = 1;
    a.item0 = 0;
    a.tiles = 0;
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
