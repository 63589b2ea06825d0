/* g53h_emm.hip - products of sorted rows with their experts' matrices in fp32, bf16 and fp16, of any sizes, and their
 * gradients (g53h_sorted_mm, g53h_sorted_mm_grad, g53h_sorted_swiglu_grad). For the rows r of expert e:
 *
 *     forward     gu[r] = W[e] . x[r],  ys[r] = gu[r] or silu(min(gate, limit)) * clip(up, -limit, limit)
 *     rows        dx[r] = W[e]^T . dys[r]
 *     matrices    dW[e] = sum over the expert's rows of dys[r] x[r]^T, zeros for an expert without rows
 */
#include <hip/hip_runtime.h>
#include <type_traits>

#include "g53h.h"
#include "g53h_elem.h"
#include "g53h_mmtile.h"
#include "g53h_runtime.h"

#define G53_EM_MAXE 1024
#define G53_EM_MAXD (1 << 24)           /* rows and columns of a matrix */

enum { G53_EM_FWD, G53_EM_ROWS, G53_EM_MATS };

struct G53EmArgs {
    const uint8_t *x;                   /* forward: rows or tokens; matrices' gradient: the same */
    const uint8_t *dy;                  /* gradients: [n][rows]                                  */
    const uint8_t *w;                   /* [NE][rows][cols]                                      */
    void *out, *gu;                     /* gu: forward with SwiGLU, or NULL                      */
    const int *offsets, *pair;          /* pair NULL: x is sorted rows                           */
    int NE, rows, cols, half;           /* half: result columns forward                          */
    float limit;                        /* SwiGLU clamp, 0 without                               */
    int w_f32, add;                     /* matrices' gradient: fp32, added to what is there      */
    int across, down;                   /* tiles across a row of results; of a matrix's rows     */
    G53Div topk;
    long wg0;                           /* first workgroup of the launch                         */
};

/* One tile of OP. DMA: operand rows start at multiples of 16 bytes and are whole pieces. */
template <typename E, int OP, int WR, int WC, int MT, int NT, int NS, bool DMA>
__global__ void __launch_bounds__(64 * WR * WC, 2) k_emm(G53EmArgs a)
{
    constexpr int NW = WR * WC, BM = 16 * MT * WR, BN = 16 * NT * WC, SLOT = (BM + BN) * 128, KE = 128 / sizeof(E);
    constexpr int IA = BM / (8 * NW), IB = BN / (8 * NW), STEPS = KE / 32;
    constexpr bool AX = OP == G53_EM_MATS, BX = OP != G53_EM_FWD;       /* operand across the summed dimension */
    static_assert(IA * 8 * NW == BM && IB * 8 * NW == BN && (DMA || NS == 2), "whole instructions");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wv / WC, wc = wv % WC;
    const long wg = a.wg0 + blockIdx.x;
    const bool sw = OP == G53_EM_FWD && a.limit > 0.0f;
    const int cut = sw ? BN / 2 : BN;                                   /* result columns of a tile */
    G53Item it;
    int m0 = 0;                                                         /* first matrix row of a dW tile */
    if constexpr (OP == G53_EM_MATS) {
        const int per = a.across * a.down;
        const long total = (long)a.NE * per;
        const int run = total >= 256 ? 32 : total >= 16 ? (int)(total / 8) : 1;
        const long i = wg >> 3, item = ((i / run) * 8 + (wg & 7)) * run + i % run;
        if (item >= total) return;
        it.e = (int)(item / per);
        const int in = (int)(item % per), g = in / (8 * a.across), in_g = in % (8 * a.across);
        const int of = a.down - 8 * g < 8 ? a.down - 8 * g : 8;
        m0 = (8 * g + in_g % of) * BM;
        it.n = in_g / of;
        it.first = g53_uniform_load(a.offsets + it.e);
        it.last = g53_uniform_load(a.offsets + it.e + 1);
    } else {
        if (!g53_tile_item(a.offsets, a.NE, BM, a.across, wg, it)) return;
    }
    const int n0 = it.n * cut, live = it.last - it.first;
    if (OP == G53_EM_MATS && a.add && !live) return;
    const long K = OP == G53_EM_FWD ? a.cols : OP == G53_EM_ROWS ? a.rows : live;
    const int chunks = (int)((K + KE - 1) / KE);
    const uint8_t *we = a.w + (long)it.e * a.rows * a.cols * sizeof(E);
    /* token of a sorted row */
    auto token = [&](int r) -> long {
        if (!a.pair) return r;
        return g53_div(a.pair[r], a.topk);
    };

    /* along: a row's address and what the lane takes of its chunks; across: the lane's row of a chunk and its columns */
    const int u8 = (lane & 7) ^ (lane >> 3);
    const uint8_t *pa[IA], *pb[IB];
    if constexpr (!AX) {
#pragma unroll
        for (int i = 0; i < IA; i++) {
            const int r = (i * NW + wv) * 8 + (lane >> 3), s = it.first + (r < live ? r : live - 1);
            if constexpr (OP == G53_EM_FWD) pa[i] = a.x + token(s) * a.cols * sizeof(E) + u8 * 16;
            else pa[i] = a.dy + (long)s * a.rows * sizeof(E) + u8 * 16;
        }
    }
    if constexpr (!BX) {
#pragma unroll
        for (int i = 0; i < IB; i++) {
            const int r = (i * NW + wv) * 8 + (lane >> 3);
            int at = n0 + r, up = 0;
            if (sw) {               /* a wave's first half of tiles: gate, the others: up */
                const int w = r / (16 * NT), t = r / 16 % NT;
                up = t >= NT / 2;
                at = n0 + w * (8 * NT) + (up ? t - NT / 2 : t) * 16 + r % 16;
            }
            at = at < a.half ? at : a.half - 1;
            pb[i] = we + (long)(at + (up ? a.half : 0)) * a.cols * sizeof(E) + u8 * 16;
        }
    }
    auto piece_a = [&](int i, int c) -> G53Piece {
        if constexpr (!AX) {
            const long at = (long)c * 128;
            return {pa[i] + at, K * (long)sizeof(E) - at - u8 * 16};
        } else {
            typedef G53Across<E, BM, MT> X;
            const int q = (i * NW + wv) * 64 + lane, k = q / X::U, u = (q % X::U) ^ X::place(k), col = m0 * (int)sizeof(E) + u * 16;
            const int kk = c * KE + k;
            return {a.dy + ((long)(it.first + kk) * a.rows * sizeof(E) + col), kk < live ? (long)a.rows * (long)sizeof(E) - col : 0};
        }
    };
    auto piece_b = [&](int i, int c) -> G53Piece {
        if constexpr (!BX) {
            const long at = (long)c * 128;
            return {pb[i] + at, K * (long)sizeof(E) - at - u8 * 16};
        } else {
            typedef G53Across<E, BN, NT> X;
            const int q = (i * NW + wv) * 64 + lane, k = q / X::U, u = (q % X::U) ^ X::place(k);
            const long col = (long)n0 * sizeof(E) + u * 16, kk = (long)c * KE + k, end = (long)a.cols * sizeof(E) - col;
            if constexpr (OP == G53_EM_ROWS) {
                return {we + (kk * a.cols * (long)sizeof(E) + col), kk < K ? end : 0};
            } else {
                /* the instruction's rows of x, asked for as scalars: their counter is not the loads' */
                constexpr int ROWS = 64 / X::U > 0 ? 64 / X::U : 1;
                const int k0 = c * KE + (i * NW + wv) * 64 / X::U;
                long t = 0;
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    const int s = it.first + (k0 + r < live ? k0 + r : live - 1);
                    const long tr = a.pair ? g53_div(g53_uniform_load(a.pair + s), a.topk) : s;
                    t = lane / X::U == r || ROWS == 1 ? tr : t;
                }
                return {a.x + (t * a.cols * (long)sizeof(E) + col), kk < live ? end : 0};
            }
        }
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    auto ask = [&](int c, int slot) {
        const uint32_t to = lds0 + slot * SLOT + wv * 1024;
#pragma unroll
        for (int i = 0; i < IA; i++) {
            const G53Piece s = piece_a(i, c);
            g53_to_lds(s.n > 0 ? s.p : (const uint8_t *)&g53_nothing, to + i * NW * 1024);
        }
#pragma unroll
        for (int i = 0; i < IB; i++) {
            const G53Piece s = piece_b(i, c);
            g53_to_lds(s.n > 0 ? s.p : (const uint8_t *)&g53_nothing, to + BM * 128 + i * NW * 1024);
        }
    };
    g53_v4w ra[DMA ? 1 : IA], rb[DMA ? 1 : IB];
    auto fetch = [&](int c) {
        if constexpr (!DMA) {
#pragma unroll
            for (int i = 0; i < IA; i++) ra[i] = g53_piece<E>(piece_a(i, c));
#pragma unroll
            for (int i = 0; i < IB; i++) rb[i] = g53_piece<E>(piece_b(i, c));
        }
    };
    auto put = [&](int slot) {
        if constexpr (!DMA) {
            uint8_t *to = lds + slot * SLOT + wv * 1024 + lane * 16;
#pragma unroll
            for (int i = 0; i < IA; i++) *(g53_v4w *)(to + i * NW * 1024) = ra[i];
#pragma unroll
            for (int i = 0; i < IB; i++) *(g53_v4w *)(to + BM * 128 + i * NW * 1024) = rb[i];
        }
    };

    typedef G53Along<E> Al;
    typename std::conditional<AX, G53Across<E, BM, MT>, Al>::type fa;
    typename std::conditional<BX, G53Across<E, BN, NT>, Al>::type fb;
    fa.setup(wr * 16 * MT);
    fb.setup(wc * 16 * NT);
    g53_v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[m][t] = (g53_v4f){0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](int slot) {
        const uint8_t *la = lds + slot * SLOT, *lb = la + BM * 128;
#pragma unroll
        for (int j = 0; j < STEPS; j++) {
            G53Frag<E> b[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) fb.read(b[t], lb, t, j);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                G53Frag<E> v;
                fa.read(v, la, m, j);
#pragma unroll
                for (int t = 0; t < NT; t++) acc[m][t] = g53_mm<E>(b[t], v, acc[m][t]);
            }
        }
    };
    if constexpr (DMA) {
        const int ahead = chunks < NS - 1 ? chunks : NS - 1;
        for (int c = 0; c < ahead; c++) ask(c, c);
        int slot = 0;
        for (int c = 0; c < chunks; c++) {
            /* chunks behind c that are on their way: NS - 2, less at the end */
            if (c + NS - 2 < chunks) g53_loads_left<(NS - 2) * (IA + IB)>();
            else g53_loads_left<0>();
            g53_meet();
            const int next = slot == 0 ? NS - 1 : slot - 1;             /* the slot of chunk c - 1 */
            if (c + NS - 1 < chunks) ask(c + NS - 1, next);
            multiply(slot);
            slot = slot == NS - 1 ? 0 : slot + 1;
        }
    } else {
        if (chunks) {
            fetch(0);
            put(0);
        }
        for (int c = 0; c < chunks; c++) {
            __syncthreads();
            if (c + 1 < chunks) fetch(c + 1);
            multiply(c & 1);
            if (c + 1 < chunks) put(c + 1 & 1);
        }
    }

    /* lane (m, q) of a tile: columns 4 q .. 4 q + 3 of row m */
    const int m = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int r = (wr * MT + i) * 16 + m;
        if constexpr (OP == G53_EM_MATS) {
            if (m0 + r >= a.rows) continue;
            const long at = ((long)it.e * a.rows + m0 + r) * a.cols;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int c = n0 + (wc * NT + t) * 16 + 4 * q;
                if (a.w_f32) g53_store4((float *)a.out + at, c, a.cols, acc[i][t], a.add);
                else g53_store4((E *)a.out + at, c, a.cols, acc[i][t], a.add);
            }
        } else {
            if (r >= live) continue;
            const long s = it.first + r;
            if (OP == G53_EM_ROWS || !sw) {
                const int N = OP == G53_EM_ROWS ? a.cols : a.half;
#pragma unroll
                for (int t = 0; t < NT; t++)
                    g53_store4((E *)a.out + s * N, n0 + (wc * NT + t) * 16 + 4 * q, N, acc[i][t], false);
            } else {
#pragma unroll
                for (int t = 0; t < NT / 2; t++) {
                    const int c = n0 + (wc * NT / 2 + t) * 16 + 4 * q;
                    g53_v4f v;
#pragma unroll
                    for (int k = 0; k < 4; k++) v[k] = g53_swiglu1(acc[i][t][k], acc[i][t + NT / 2][k], a.limit);
                    g53_store4((E *)a.out + s * a.half, c, a.half, v, false);
                    if (a.gu) {
                        g53_store4((E *)a.gu + s * a.rows, c, a.half, acc[i][t], false);
                        g53_store4((E *)a.gu + s * a.rows + a.half, c, a.half, acc[i][t + NT / 2], false);
                    }
                }
            }
        }
    }
}

/* Threads of a launch are counted in 32 bits. */
#define G53_EM_WGS (1l << 22)

template <typename E, int OP, int WR, int WC, int MT, int NT, int NS, bool DMA> static int launch(G53EmArgs a, long n)
{
    constexpr int BM = 16 * MT * WR, BN = 16 * NT * WC;
    constexpr size_t LDS = (size_t)NS * (BM + BN) * 128;
    static int allowed = 0;
    if (!allowed) {
        G53_TRY(hipFuncSetAttribute((const void *)k_emm<E, OP, WR, WC, MT, NT, NS, DMA>,
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS));
        allowed = 1;
    }
    const int N = OP == G53_EM_FWD ? a.half : a.cols, cut = OP == G53_EM_FWD && a.limit > 0.0f ? BN / 2 : BN;
    a.across = (N + cut - 1) / cut;
    a.down = (a.rows + BM - 1) / BM;
    const long most = a.NE < n ? a.NE : n;              /* experts that can have rows */
    const long items = OP == G53_EM_MATS ? (long)a.NE * a.down * a.across : (n / BM + most) * a.across;
    const long wgs = (items + 7) / 8 * 8 + (items < 8 ? 8 : items < 256 ? (items + 7) / 8 * 8 : 256);   /* whole runs on every die */
    for (long w0 = 0; w0 < wgs; w0 += G53_EM_WGS) {
        a.wg0 = w0;
        const dim3 grid((unsigned)(wgs - w0 < G53_EM_WGS ? wgs - w0 : G53_EM_WGS));
        hipLaunchKernelGGL((k_emm<E, OP, WR, WC, MT, NT, NS, DMA>), grid, dim3(64 * WR * WC), LDS, g53h_stream(), a);
        G53_LAUNCHED("k_emm");
    }
    return 0;
}

template <typename E, int OP> static int by_size(const G53EmArgs &a, long n)
{
    /* whole pieces of 16 bytes at multiples of 16 */
    const uintptr_t at = OP == G53_EM_FWD ? (uintptr_t)a.x | (uintptr_t)a.w
                         : OP == G53_EM_ROWS ? (uintptr_t)a.dy | (uintptr_t)a.w : (uintptr_t)a.dy | (uintptr_t)a.x;
    const size_t odd = (a.cols * sizeof(E)) | (OP == G53_EM_FWD ? 0 : a.rows * sizeof(E));
    if ((at | odd) & 15) return launch<E, OP, 2, 2, 4, 4, 2, false>(a, n);
    return launch<E, OP, 2, 2, 4, 4, 2, true>(a, n);
}

/* ------------------------------------------------------------- SwiGLU's gradient ---- */
/* dgu of dact and gu, eight elements of gate and of up a thread; a workgroup's rows by `chunks` of 2048. */
template <typename E>
__global__ void __launch_bounds__(256) k_swiglu_grad(E *dgu, const E *dact, const E *gu, const int *__restrict__ end, int H,
                                                     int chunks, float limit, long wg0)
{
    const long wg = wg0 + blockIdx.x, r = wg / chunks;
    const int c = ((int)(wg % chunks) * 256 + threadIdx.x) * 8;
    if (c >= H || r >= *end) return;
    float d[8], g[8], u[8];
    g53_load8_to(d, dact + r * H, c, H);
    g53_load8_to(g, gu + r * 2 * H, c, H);
    g53_load8_to(u, gu + r * 2 * H + H, c, H);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float gc = g[i] > limit ? limit : g[i], uc = u[i] > limit ? limit : (u[i] < -limit ? -limit : u[i]);
        const float x = expf(-fabsf(gc)), s = (gc >= 0.0f ? 1.0f : x) / (1.0f + x);      /* no overflow: small, not zero */
        const float dg = d[i] * uc * s * (1.0f + gc * (1.0f - s)), du = d[i] * gc * s;
        const bool g_out = g[i] > limit, u_out = u[i] > limit || u[i] < -limit;
        g[i] = g_out ? 0.0f : dg;
        u[i] = u_out ? 0.0f : du;
    }
    g53_store8_to(dgu + r * 2 * H, g, c, H);
    g53_store8_to(dgu + r * 2 * H + H, u, c, H);
}

/* --------------------------------------------------------------------- the calls ---- */
static int em_plan(const char *who, const G53hSort *p, int dt, int rows, int cols, G53EmArgs &a)
{
    if (!p || p->T < 0 || p->topk < 1 || p->topk > 64 || p->n_experts < 1 || p->n_experts > G53_EM_MAXE ||
        (long)p->T * p->topk > 0x7fffffffl || !p->offsets || (p->T && !p->pair))
        return g53h_fail("%s: no plan of g53h_sort_tokens", who);
    if (!g53_elem_bytes(dt)) return g53h_fail("%s: element type %d", who, dt);
    if (rows < 1 || rows > G53_EM_MAXD || cols < 1 || cols > G53_EM_MAXD)
        return g53h_fail("%s: matrices of %d x %d (1 to 2^24 rows and columns)", who, rows, cols);
    a = G53EmArgs{};
    a.offsets = p->offsets;
    a.NE = p->n_experts;
    a.topk = g53_div_of(p->topk);
    a.rows = rows;
    a.cols = cols;
    a.half = rows;
    return 0;
}

static int em_aligned(const char *who, int dt, const void *p)
{
    return (uintptr_t)p & (g53_elem_bytes(dt) - 1) ? g53h_fail("%s: addresses must be multiples of an element", who) : 0;
}

extern "C" int g53h_sorted_mm(void *ys, void *gu, const void *x, int dt, int gather, const G53hSort *p, const void *w,
                              int rows, int cols, float swiglu_limit)
{
    const char *who = "g53h_sorted_mm";
    G53EmArgs a;
    if (em_plan(who, p, dt, rows, cols, a)) return -1;
    if (!(swiglu_limit >= 0.0f) || swiglu_limit > 3.0e38f) return g53h_fail("%s: SwiGLU limit %g", who, swiglu_limit);
    if (swiglu_limit > 0.0f && rows % 2) return g53h_fail("%s: SwiGLU of %d rows", who, rows);
    if (gu && !(swiglu_limit > 0.0f)) return g53h_fail("%s: gate and up without SwiGLU", who);
    if (!p->T) return 0;
    if (!ys || !x || !w) return g53h_fail("%s: no rows or no matrices", who);
    if (em_aligned(who, dt, ys) || em_aligned(who, dt, gu) || em_aligned(who, dt, x) || em_aligned(who, dt, w)) return -1;
    if (g53h_ready()) return -1;
    a.x = (const uint8_t *)x;
    a.w = (const uint8_t *)w;
    a.out = ys;
    a.gu = gu;
    a.pair = gather ? p->pair : nullptr;
    a.limit = swiglu_limit;
    if (swiglu_limit > 0.0f) a.half = rows / 2;
    int rc;
    G53_BY_TYPE(dt, rc = (by_size<E, G53_EM_FWD>(a, (long)p->T * p->topk)));
    return rc;
}

extern "C" int g53h_sorted_mm_grad(void *dx, void *dw, int dw_dt, int add, const void *dys, const void *x, int dt, int gather,
                                   const G53hSort *p, const void *w, int rows, int cols)
{
    const char *who = "g53h_sorted_mm_grad";
    G53EmArgs a;
    if (em_plan(who, p, dt, rows, cols, a)) return -1;
    if (!dx && !dw) return g53h_fail("%s: neither gradient wanted", who);
    if (dw && dw_dt != dt && dw_dt != G53H_F32) return g53h_fail("%s: matrices' gradient of type %d", who, dw_dt);
    if (p->T && (!dys || (dx && !w) || (dw && !x))) return g53h_fail("%s: no rows or no matrices", who);
    if (em_aligned(who, dt, dys) || em_aligned(who, dt, dx) || em_aligned(who, dt, x) || em_aligned(who, dt, w) ||
        (dw && em_aligned(who, dw_dt, dw)))
        return -1;
    if (g53h_ready()) return -1;
    const long n = (long)p->T * p->topk;
    a.x = (const uint8_t *)x;
    a.dy = (const uint8_t *)dys;
    a.w = (const uint8_t *)w;
    int rc = 0;
    if (dx && n) {
        a.out = dx;
        G53_BY_TYPE(dt, rc = (by_size<E, G53_EM_ROWS>(a, n)));
    }
    if (!rc && dw) {
        a.out = dw;
        a.pair = gather ? p->pair : nullptr;
        a.w_f32 = dw_dt == G53H_F32;
        a.add = add != 0;
        G53_BY_TYPE(dt, rc = (by_size<E, G53_EM_MATS>(a, n)));
    }
    return rc;
}

extern "C" int g53h_sorted_swiglu_grad(void *dgu, const void *dact, const void *gu, int dt, int inter, const G53hSort *p,
                                       float limit)
{
    const char *who = "g53h_sorted_swiglu_grad";
    G53EmArgs a;
    if (em_plan(who, p, dt, inter, 1, a)) return -1;
    if (!(limit > 0.0f) || limit > 3.0e38f) return g53h_fail("%s: SwiGLU limit %g", who, limit);
    if (!p->T) return 0;
    if (!dgu || !dact || !gu) return g53h_fail("%s: no rows", who);
    if (em_aligned(who, dt, dgu) || em_aligned(who, dt, dact) || em_aligned(who, dt, gu)) return -1;
    if (g53h_ready()) return -1;
    const int chunks = (inter + 2047) / 2048;
    const long total = (long)p->T * p->topk * chunks, most = 1l << 23;
    for (long w0 = 0; w0 < total; w0 += most) {
        const unsigned wgs = (unsigned)(total - w0 < most ? total - w0 : most);
        G53_BY_TYPE(dt, hipLaunchKernelGGL(k_swiglu_grad<E>, dim3(wgs), dim3(256), 0, g53h_stream(), (E *)dgu, (const E *)dact,
                                           (const E *)gu, p->offsets + p->n_experts, inter, chunks, limit, w0));
        G53_LAUNCHED("k_swiglu_grad");
    }
    return 0;
}
