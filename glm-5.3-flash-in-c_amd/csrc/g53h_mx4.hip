/* g53h_mx4.hip - microscaled 4-bit matrices: E2M1 levels with one power of two for 32 columns of a row, the block format of
 * the scaled matrix instructions. Quantisation of rows and back, and products of two such matrices, of one matrix
 * (g53h_mm_mx4) or of the matrix of each sorted row's expert (g53h_sorted_mm_mx4).
 *
 *     y[t][r] = sum over blocks b of  2^(xs[t][b] + s[r][b] - 254) * sum over c in b of xq[t][c] q[r][c]
 *
 * Levels and scales go to v_mfma_scale_f32_16x16x128_f8f6f4 as they lie: lane (m, q) takes the 32 levels, 16 bytes, of
 * row m and block q of four, and their scale. Products and scales are exact; sums are fp32.
 *
 * Measured: 65536 x 4096 bf16 quantised in 114 us and read back in 129, 6.0 and 5.3 TB/s of what passes (a copy 4.67, a fill
 * 6.8; one behind the other, as the cache holds it, 137 and 123); gate/up 4096 x 4096 of one token's 8 of 288 experts 15.0 to
 * 18.6 us, 71 MB, HBM behind a launch and the search of a row's expert; 65536 x 4096 by 5 rows 28.6 us, 5.0 TB/s; 8192 x 8192
 * by 8192 rows 331 us, 3320 TFLOP/s, and gate/up by 4096 tokens, 8 of 64 experts, 448 us, 2450: a chunk of 256 columns is 512
 * cycles of matrix instructions beside 32 to 48 KB on their way to LDS, and waits are 33 and 41% of the waves' time (matrix
 * instructions 44 and 28% of the CUs').
 */
#include <hip/hip_runtime.h>
#include <type_traits>

#include "g53h.h"
#include "g53h_elem.h"
#include "g53h_mmtile.h"
#include "g53h_runtime.h"

#define G53_MX_MAXE 1024
#define G53_MX_MAXC (1 << 24)
#define G53_MX_WGS (1l << 22)           /* workgroups of a launch: its threads are counted in 32 bits */

typedef int g53_v8i __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(1))) G53v4w_byte { g53_v4w v; };

/* ---------------------------------------------------------------- quantisation ---- */
/* Eight columns a lane, a block in four: its largest size by DPP, the scale's exponent that of the largest value less 2
 * (6 is 1.5 * 2^2), so that levels reach 4 to 8 and those above 6 count as 6. A block with a value that is not finite has
 * the scale 255, NaN, and levels of zero. */
template <typename E>
__global__ void __launch_bounds__(256) k_mx4_quant(uint8_t *__restrict__ w, uint8_t *__restrict__ s, const E *__restrict__ x,
                                                   long eights, long wg0)
{
    const long i = (wg0 + blockIdx.x) * 256 + threadIdx.x;      /* rows are whole blocks: one run of eights */
    if (i >= eights) return;
    float v[8];
    g53_load8(v, x + i * 8);
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const unsigned u = __builtin_bit_cast(unsigned, v[k]) & 0x7fffffffu;
        top = u > top ? u : top;
    }
    unsigned o = __builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true);      /* lane ^ 1 */
    top = o > top ? o : top;
    o = __builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true);               /* lane ^ 2 */
    top = o > top ? o : top;
    const int e = (int)(top >> 23);
    const int b = e == 255 ? 255 : e > 2 ? e - 2 : 0;
    /* by 2^(127 - b), exactly: levels */
    const float up = __builtin_bit_cast(float, (unsigned)(254 - b) << 23);
    unsigned q = 0;
#define G53_PAIR(k) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2 * k] * up, v[2 * k + 1] * up, 1.0f, k)
    G53_PAIR(0); G53_PAIR(1); G53_PAIR(2); G53_PAIR(3);
#undef G53_PAIR
    if (b == 255) q = 0;
    ((unsigned *)w)[i] = q;
    if (!(threadIdx.x & 3)) s[i >> 2] = (uint8_t)b;
}

template <typename E>
__global__ void __launch_bounds__(256) k_mx4_dequant(E *__restrict__ x, const uint8_t *__restrict__ w, const uint8_t *__restrict__ s,
                                                     long eights, long wg0)
{
    const long i = (wg0 + blockIdx.x) * 256 + threadIdx.x;
    if (i >= eights) return;
    const unsigned q = ((const unsigned *)w)[i], b = s[i >> 2];
    const float up = __builtin_bit_cast(float, b == 0 ? 1u << 22 : b == 255 ? 0x7fc00000u : b << 23);
    float v[8];
#define G53_PAIR(k)                                                                       \
    do {                                                                                  \
        const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, k);              \
        v[2 * k] = p[0] * up;                                                             \
        v[2 * k + 1] = p[1] * up;                                                         \
    } while (0)
    G53_PAIR(0); G53_PAIR(1); G53_PAIR(2); G53_PAIR(3);
#undef G53_PAIR
    g53_store8(x + i * 8, v);
}

/* -------------------------------------------------------------------- products ---- */
struct G53MxArgs {
    const uint8_t *x, *xs;              /* levels [T][cols / 2] and scales [T][cols / 32] */
    const uint8_t *w, *s;               /* [NE][rows][cols / 2], [NE][rows][cols / 32]     */
    const int *offsets, *pair;          /* NULL: one matrix; x is sorted rows              */
    void *out;
    int NE, T, rows, cols, half;
    float limit;
    int across;
    G53Div topk;
    long wg0;
};

/* One tile, by the stream of k_emm (g53h_emm.hip): a chunk is 256 columns, two steps of 128. Scales come 16 a row at a time,
 * those of two chunks, through registers, which turn each quarter's four side by side: asked for in the second half of
 * an odd chunk, put down in that of the even one behind it, and read in that of the odd one behind that. */
template <typename E, int WR, int WC, int MT, int NT, int NS>
__global__ void __launch_bounds__(64 * WR * WC, 2) k_mx4(G53MxArgs a)
{
    constexpr int NW = WR * WC, BM = 16 * MT * WR, BN = 16 * NT * WC, SLOT = (BM + BN) * 128, SEG = (BM + BN) * 16;
    constexpr int IA = BM / (8 * NW), IB = BN / (8 * NW), IS = (BM + BN + 64 * NW - 1) / (64 * NW);
    static_assert(IA * 8 * NW == BM && IB * 8 * NW == BN, "whole instructions");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wv / WC, wc = wv % WC;
    const bool sw = a.limit > 0.0f;
    const int cut = sw ? BN / 2 : BN;
    G53Item it;
    const long wg = a.wg0 + blockIdx.x;
    if (a.offsets) {
        if (!g53_tile_item(a.offsets, a.NE, BM, a.across, wg, it)) return;
    } else {
        const int tiles = (int)(((unsigned)a.T + BM - 1) / BM);
        const long total = (long)tiles * a.across, item = g53_deal(wg, total);
        if (item >= total) return;
        int t;
        g53_eight(item, tiles, a.across, t, it.n);
        it.e = 0;
        it.first = t * BM;
        it.last = a.T - it.first > BM ? it.first + BM : a.T;
    }
    const int n0 = it.n * cut, live = it.last - it.first, rb = a.cols / 2, sb = a.cols / 32;
    const int chunks = (rb + 127) / 128;
    const long e0 = (long)it.e * a.rows;
    auto x_row = [&](int r) -> long {
        const int s = it.first + (r < live ? r : live - 1);
        return a.pair ? g53_div(a.pair[s], a.topk) : s;
    };
    auto w_row = [&](int r) -> long {
        unsigned at = n0 + (unsigned)r, up = 0;     /* past a matrix's last row it may pass 2^31 */
        if (sw) {                       /* a wave's first half of tiles: gate, the others: up */
            const int t = r / 16 % NT;
            up = t >= NT / 2;
            at = n0 + (unsigned)(r / (16 * NT) * (8 * NT) + (up ? t - NT / 2 : t) * 16 + r % 16);
        }
        at = at < (unsigned)a.half ? at : a.half - 1;
        return e0 + at + (up ? a.half : 0);
    };
    const int u8 = (lane & 7) ^ (lane >> 3);
    const uint8_t *pa[IA], *pb[IB], *ps[IS];
#pragma unroll
    for (int i = 0; i < IA; i++) pa[i] = a.x + x_row((i * NW + wv) * 8 + (lane >> 3)) * rb + u8 * 16;
#pragma unroll
    for (int i = 0; i < IB; i++) pb[i] = a.w + w_row((i * NW + wv) * 8 + (lane >> 3)) * rb + u8 * 16;
#pragma unroll
    for (int i = 0; i < IS; i++) {
        const int r = i * 64 * NW + tid;
        ps[i] = r < BM ? a.xs + x_row(r) * sb : a.s + w_row(r - BM < BN ? r - BM : BN - 1) * sb;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    /* Behind a row's end its last piece comes again: levels are finite whatever they are, and both scales there are 0, so what
     * they add is below fp32's steps. */
    const int end = rb - 16 - u8 * 16;
    int off = 0;
    auto to_chunk = [&](int c) { off = c * 128 < end ? c * 128 : end; };
    auto ask1 = [&](int slot, int i) {
        const uint32_t to = lds0 + slot * SLOT + wv * 1024;
        g53_to_lds((i < IA ? pa[i < IA ? i : 0] : pb[i < IA ? 0 : i - IA]) + off,
                   to + (i < IA ? i * NW * 1024 : BM * 128 + (i - IA) * NW * 1024));
    };
    g53_v4w rs[IS];
    auto fetch = [&](int seg) {
        const int n = sb - seg * 16;
#pragma unroll
        for (int i = 0; i < IS; i++) {
            const uint8_t *p = ps[i] + (long)seg * 16;
            if (n >= 16) rs[i] = ((const G53v4w_byte *)p)->v;
            else
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    unsigned v = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) v |= 4 * k + j < n ? (unsigned)p[4 * k + j] << 8 * j : 0u;
                    rs[i][k] = v;
                }
        }
    };
    uint8_t *const lds_s = lds + NS * SLOT;
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < IS; i++) {
            const int r = i * 64 * NW + tid;
            const unsigned l0 = __builtin_amdgcn_perm(rs[i][1], rs[i][0], 0x05010400u), l1 = __builtin_amdgcn_perm(rs[i][1], rs[i][0], 0x07030602u);
            const unsigned h0 = __builtin_amdgcn_perm(rs[i][3], rs[i][2], 0x05010400u), h1 = __builtin_amdgcn_perm(rs[i][3], rs[i][2], 0x07030602u);
            const g53_v4w o = {__builtin_amdgcn_perm(h0, l0, 0x05040100u), __builtin_amdgcn_perm(h0, l0, 0x07060302u),
                               __builtin_amdgcn_perm(h1, l1, 0x05040100u), __builtin_amdgcn_perm(h1, l1, 0x07060302u)};
            if (r < BM + BN) *(g53_v4w *)(lds_s + buf * SEG + r * 16) = o;
        }
    };
    const int m = lane & 15, q = lane >> 4;
    const int fa = (wr * 16 + m) * 128 + ((q ^ (m & 7)) << 4), fb = BM * 128 + (wc * 16 * NT + m) * 128 + ((q ^ (m & 7)) << 4);
    const int sa = (wr * 16 + m) * 16 + 4 * q, sw_at = (BM + wc * 16 * NT + m) * 16 + 4 * q;
    g53_v4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[i][t] = (g53_v4f){0.0f, 0.0f, 0.0f, 0.0f};
    auto run = [&](auto M_) {
        constexpr int M = decltype(M_)::value;              /* row tiles of a wave that are there */
        constexpr int RD = (M + NT + M - 1) / M, IM = IA * M / MT > 0 ? IA * M / MT : 1, AD = (IM + IB + M - 1) / M;
        g53_v4w va[2][M], vb[2][NT];
        int xs[M], ws[NT];
        auto read1 = [&](int to, int slot, int j, int i) {
            const uint8_t *l = lds + slot * SLOT;
            if (i < NT) vb[to][i] = *(const g53_v4w *)(l + (fb ^ j * 64) + i * 2048);
            else va[to][i - NT] = *(const g53_v4w *)(l + (fa ^ j * 64) + (i - NT) * (WR * 2048));
        };
        auto scale_x = [&](int buf, int i) { xs[i] = *(const int *)(lds_s + buf * SEG + sa + i * (WR * 256)); };
        auto scale_w = [&](int buf) {
#pragma unroll
            for (int t = 0; t < NT; t++) ws[t] = *(const int *)(lds_s + buf * SEG + sw_at + t * 256);
        };
#define G53_MX_ROW(i, h, byte)                                                                                          \
    _Pragma("unroll") for (int t = 0; t < NT; t++) {                                                                    \
        const g53_v8i b = {(int)vb[h][t][0], (int)vb[h][t][1], (int)vb[h][t][2], (int)vb[h][t][3], 0, 0, 0, 0};        \
        const g53_v8i v = {(int)va[h][i][0], (int)va[h][i][1], (int)va[h][i][2], (int)va[h][i][3], 0, 0, 0, 0};        \
        acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, v, acc[i][t], 4, 4, byte, ws[t], byte, xs[i]); \
    }                                                                                                                   \
    __builtin_amdgcn_sched_barrier(0)
        fetch(0);
        put(0);
#pragma unroll
        for (int c = 0; c < NS; c++) {
            to_chunk(c);
#pragma unroll
            for (int i = 0; i < IM + IB; i++) ask1(c, i < IM ? i : i - IM + IA);
        }
        fetch(1);
        g53_loads_left<0>();
        g53_meet();
#pragma unroll
        for (int i = 0; i < M + NT; i++) read1(0, 0, 0, i);
#pragma unroll
        for (int i = 0; i < M; i++) scale_x(0, i);
        scale_w(0);
        int slot = 0;
        auto chunk = [&](int c, auto odd_) {
            constexpr int odd = decltype(odd_)::value;
            const int next = slot == NS - 1 ? 0 : slot + 1;
#pragma unroll
            for (int i = 0; i < M; i++) {
#pragma unroll
                for (int k = i * RD; k < (i + 1) * RD && k < M + NT; k++) read1(1, slot, 1, k);
                G53_MX_ROW(i, 0, 2 * odd);
            }
            g53_loads_left<(NS - 2) * (IM + IB)>();
            g53_meet();
            to_chunk(c + NS);
            if (odd) fetch((c + 1) / 2 + 1);
            else put((c / 2 + 1) & 1);
#pragma unroll
            for (int i = 0; i < M; i++) {
#pragma unroll
                for (int k = i * AD; k < (i + 1) * AD && k < IM + IB; k++) ask1(slot, k < IM ? k : k - IM + IA);
#pragma unroll
                for (int k = i * RD; k < (i + 1) * RD && k < M + NT; k++) read1(0, next, 0, k);
                G53_MX_ROW(i, 1, 2 * odd + 1);
                if (odd) scale_x((c + 1) / 2 & 1, i);       /* the next segment's, each in the place of the one just used */
            }
            if (odd) scale_w((c + 1) / 2 & 1);
            slot = next;
        };
        for (int c = 0;; c += 2) {
            chunk(c, std::integral_constant<int, 0>{});
            if (c + 1 >= chunks) break;
            chunk(c + 1, std::integral_constant<int, 1>{});
            if (c + 2 >= chunks) break;
        }
#undef G53_MX_ROW
        g53_loads_left<0>();                                /* no load outlives the workgroup's LDS */
    };
    if constexpr (MT < 4) run(std::integral_constant<int, MT>{});
    else if (live <= BM / 4) run(std::integral_constant<int, MT / 4>{});
    else if (live <= BM / 2) run(std::integral_constant<int, MT / 2>{});
    else run(std::integral_constant<int, MT>{});
    g53_meet();
    uint8_t *const buf = lds + wv * (MT * NT * 256 * (int)sizeof(E));
    const int r0 = wr * 16;
    const long c = n0 + (long)(wc * (sw ? NT / 2 : NT) * 16);
    const int most = (int)(a.half - c);
    E *at = (E *)a.out + (it.first + (long)r0) * a.half + c;
    if (!sw) {
        g53_leave<E, WR>(buf, at, a.half, acc, live - r0, most);
    } else {
        g53_v4f v[MT][NT / 2];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int t = 0; t < NT / 2; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) v[i][t][k] = g53_swiglu1<E>(acc[i][t][k], acc[i][t + NT / 2][k], a.limit);
        g53_leave<E, WR>(buf, at, a.half, v, live - r0, most);
    }
}

template <typename E, int WR, int WC, int MT, int NT, int NS> static int launch(G53MxArgs a, long n)
{
    constexpr int BM = 16 * MT * WR, BN = 16 * NT * WC;
    constexpr size_t LDS = (size_t)(BM + BN) * (NS * 128 + 2 * 16);
    static_assert(LDS >= WR * WC * MT * NT * 256 * sizeof(E), "rows on their way out");
    static int allowed = 0;
    if (!allowed) {
        G53_TRY(hipFuncSetAttribute((const void *)k_mx4<E, WR, WC, MT, NT, NS>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS));
        allowed = 1;
    }
    const int cut = a.limit > 0.0f ? BN / 2 : BN;
    a.across = (int)(((long)a.half + cut - 1) / cut);
    const long wgs = g53_deal_wgs((a.offsets ? n / BM + (a.NE < n ? a.NE : n) : (n + BM - 1) / BM) * a.across);
    for (long w0 = 0; w0 < wgs; w0 += G53_MX_WGS) {
        a.wg0 = w0;
        const dim3 grid((unsigned)(wgs - w0 < G53_MX_WGS ? wgs - w0 : G53_MX_WGS));
        hipLaunchKernelGGL((k_mx4<E, WR, WC, MT, NT, NS>), grid, dim3(64 * WR * WC), LDS, g53h_stream(), a);
        G53_LAUNCHED("k_mx4");
    }
    return 0;
}

/* --------------------------------------------------------------------- the calls ---- */
static int mx_bad(const char *who, const G53hMx4 *m)
{
    if (!m) return g53h_fail("%s: no matrix", who);
    if (m->rows < 0 || m->cols < 32 || m->cols > G53_MX_MAXC || m->cols % 32)
        return g53h_fail("%s: %d x %d levels (columns a multiple of 32, at most 2^24)", who, m->rows, m->cols);
    if (m->rows && (!m->w || !m->s)) return g53h_fail("%s: unbound matrix", who);
    if ((uintptr_t)m->w & 15) return g53h_fail("%s: levels must start at a multiple of 16 bytes", who);
    return 0;
}

extern "C" int g53h_mx4_quant(const G53hMx4 *m, const void *x, int dt)
{
    const char *who = "g53h_mx4_quant";
    if (mx_bad(who, m)) return -1;
    if (!g53_elem_bytes(dt)) return g53h_fail("%s: element type %d", who, dt);
    if (!m->rows) return 0;
    if (!x || ((uintptr_t)x & (g53_elem_bytes(dt) - 1))) return g53h_fail("%s: no rows, or not at a multiple of an element", who);
    if (g53h_ready()) return -1;
    const long eights = (long)m->rows * m->cols / 8, wgs = (eights + 255) / 256;
    for (long w0 = 0; w0 < wgs; w0 += G53_MX_WGS) {
        const dim3 grid((unsigned)(wgs - w0 < G53_MX_WGS ? wgs - w0 : G53_MX_WGS));
        G53_BY_TYPE(dt, hipLaunchKernelGGL(k_mx4_quant<E>, grid, dim3(256), 0, g53h_stream(), m->w, m->s, (const E *)x, eights, w0));
        G53_LAUNCHED("k_mx4_quant");
    }
    return 0;
}

extern "C" int g53h_mx4_dequant(void *x, int dt, const G53hMx4 *m)
{
    const char *who = "g53h_mx4_dequant";
    if (mx_bad(who, m)) return -1;
    if (!g53_elem_bytes(dt)) return g53h_fail("%s: element type %d", who, dt);
    if (!m->rows) return 0;
    if (!x || ((uintptr_t)x & (g53_elem_bytes(dt) - 1))) return g53h_fail("%s: no rows, or not at a multiple of an element", who);
    if (g53h_ready()) return -1;
    const long eights = (long)m->rows * m->cols / 8, wgs = (eights + 255) / 256;
    for (long w0 = 0; w0 < wgs; w0 += G53_MX_WGS) {
        const dim3 grid((unsigned)(wgs - w0 < G53_MX_WGS ? wgs - w0 : G53_MX_WGS));
        G53_BY_TYPE(dt, hipLaunchKernelGGL(k_mx4_dequant<E>, grid, dim3(256), 0, g53h_stream(), (E *)x, m->w, m->s, eights, w0));
        G53_LAUNCHED("k_mx4_dequant");
    }
    return 0;
}

/* Both matrices, the type and the limit; fills what a dense and a sorted product share. */
static int mx_product(const char *who, void *y, int dt, const G53hMx4 *x, const G53hMx4 *m, float limit, G53MxArgs &a)
{
    if (mx_bad(who, x) || mx_bad(who, m)) return -1;
    if (m->rows < 1) return g53h_fail("%s: a matrix of %d rows", who, m->rows);
    if (x->cols != m->cols) return g53h_fail("%s: rows of %d columns by a matrix of %d", who, x->cols, m->cols);
    if (!g53_elem_bytes(dt)) return g53h_fail("%s: element type %d", who, dt);
    if (!(limit >= 0.0f) || limit > 3.0e38f) return g53h_fail("%s: SwiGLU limit %g", who, limit);
    if (limit > 0.0f && m->rows % 2) return g53h_fail("%s: SwiGLU of %d rows", who, m->rows);
    if ((uintptr_t)y & (g53_elem_bytes(dt) - 1)) return g53h_fail("%s: results must be at a multiple of an element", who);
    a = G53MxArgs{};
    a.x = x->w;
    a.xs = x->s;
    a.w = m->w;
    a.s = m->s;
    a.out = y;
    a.NE = 1;
    a.T = x->rows;
    a.rows = m->rows;
    a.cols = m->cols;
    a.limit = limit;
    a.half = limit > 0.0f ? m->rows / 2 : m->rows;
    a.topk = g53_div_of(1);
    return 0;
}

/* Tiles by the rows that experts have, all alike, as in g53h_emm.hip. us, bf16, tiles of 128 x 128, 64 x 128, 32 x 128 (of
 * 256 x 128, one workgroup of four waves a CU, more than any; of 128 x 256, eight waves and three slots, 152 and 90 for the first
 * two, 328 for 8192 rows, 32 for 512):
 *     4096 x 4096, 64 experts, top-8: 1024 tokens 158 210 255, 256 93 98 105, 16 55 54 62, 1 18.5 18.3 18.0
 *     1024 x 1024, 16 experts, top-4: 1024 tokens 12 16 16, 64 6.5 6.4 5.8
 *     8192 x 8192: 8192 rows 349 503 661, 512 30 31 48, 64 24 24 22, 1 20.6 20.4 20.5
 * The tests repeat this rule, to name the tile that a size takes. */
template <typename E> static int by_size(const G53MxArgs &a, long n)
{
    const long busy = a.offsets ? (a.NE < n ? a.NE : n) : 1, mean = (n + busy - 1) / busy, cus = g53h_num_cus();
    auto tiles = [&](int bm, int bn) { return (a.offsets ? n / bm + busy : (n + bm - 1) / bm) * (((long)a.rows + bn - 1) / bn); };
    if (mean >= 32 && tiles(128, 256) >= 2 * cus) return launch<E, 2, 4, 4, 4, 3>(a, n);
    if (mean >= 32 && tiles(128, 128) >= cus) return launch<E, 2, 2, 4, 4, 2>(a, n);
    if (mean > 1 && tiles(64, 128) >= 2 * cus) return launch<E, 1, 4, 4, 2, 2>(a, n);
    return launch<E, 1, 4, 2, 2, 2>(a, n);
}

extern "C" int g53h_mm_mx4(void *y, int dt, const G53hMx4 *x, const G53hMx4 *m, float swiglu_limit)
{
    G53MxArgs a;
    if (mx_product("g53h_mm_mx4", y, dt, x, m, swiglu_limit, a)) return -1;
    if (!a.T) return 0;
    if (!y) return g53h_fail("g53h_mm_mx4: no results");
    if (g53h_ready()) return -1;
    int rc;
    G53_BY_TYPE(dt, rc = by_size<E>(a, a.T));
    return rc;
}

extern "C" int g53h_sorted_mm_mx4(void *ys, int dt, const G53hMx4 *x, int gather, const G53hSort *p, const G53hMx4 *m,
                                  float swiglu_limit)
{
    const char *who = "g53h_sorted_mm_mx4";
    G53MxArgs a;
    if (mx_product(who, ys, dt, x, m, swiglu_limit, a)) return -1;
    if (!p || p->T < 0 || p->topk < 1 || p->topk > 64 || p->n_experts < 1 || p->n_experts > G53_MX_MAXE ||
        (long)p->T * p->topk > 0x7fffffffl || !p->offsets || (p->T && !p->pair))
        return g53h_fail("%s: no plan of g53h_sort_tokens", who);
    const long n = (long)p->T * p->topk;
    if (x->rows < (gather ? p->T : n)) return g53h_fail("%s: %d rows of x, the plan has %ld", who, x->rows, gather ? (long)p->T : n);
    if (!p->T) return 0;
    if (!ys) return g53h_fail("%s: no results", who);
    if (g53h_ready()) return -1;
    a.offsets = p->offsets;
    a.pair = gather ? p->pair : nullptr;
    a.NE = p->n_experts;
    a.topk = g53_div_of(p->topk);
    int rc;
    G53_BY_TYPE(dt, rc = by_size<E>(a, n));
    return rc;
}
