/* g53h_emm.hip - products of sorted rows with their experts' matrices in fp32, bf16 and fp16, of any sizes, and their
 * gradients (g53h_sorted_mm, g53h_sorted_mm_grad, g53h_sorted_swiglu_grad). For the rows r of expert e:
 *
 *     forward     gu[r] = W[e] . x[r],  ys[r] = gu[r] or silu(min(gate, limit)) * clip(up, -limit, limit)
 *     rows        dx[r] = W[e]^T . dys[r]
 *     matrices    dW[e] = sum over the expert's rows of dys[r] x[r]^T, zeros for an expert without rows
 *
 * A tile of results belongs to one expert; a workgroup finds its tile from the plan's offsets, so the host need not know how
 * many rows an expert has. Operands stream through LDS (g53h_mmtile.h); products are v_mfma_f32_16x16x32 of bf16 or fp16 with
 * fp32 sums, the matrix's rows as the first operand, so that a lane holds four neighbours of a result's row. With 16 bits the
 * operands of a step of 32 leave LDS while those before it are multiplied. fp32 enters as three bf16 planes, six products
 * each: at the rates of large library products 2.4e14 a second against 1.45e14 of the fp32 matrix instructions. Splitting takes
 * vector work of about the products' time, and what is reached is no more than the latter: 1.4e14 by 2048 tokens.
 *
 * Measured (bf16 unless named; a 4 GiB copy moves 4.67 TB/s, a library product of 8192 cubed 1448 TFLOP/s in bf16 with both
 * operands along the summed dimension, 145 in fp32):
 *     8192 x 8192 by 8192 rows: forward 858 us, 1282 TFLOP/s, bound by power and LDS; rows 1005, 1094; matrices 1257, 875
 *     gate/up 4096 x 4096 of one token's 8 of 288 experts, SwiGLU: 52 to 55 us, 4.9 to 5.2 TB/s, HBM
 *     the same by 4096 tokens, 8 of 64, gate and up kept: 1137 to 1160 us, 950 to 967 TFLOP/s (rows of popular experts 2000, of
 *     others none: tiles partly empty, dies unevenly loaded at the end)
 *     gradients of 2048 such tokens, matrices in fp32: SwiGLU 65 us (5.2 TB/s), rows 752, matrices 1446; the last write 4.3 GB,
 *     which alone take 870, and sum some 400 rows each between: instructions of addresses and of the way out, 5 beside a matrix
 *     instruction. Added to what is there, element by element: 2679
 *     fp16 1001 x 1023, 301 tokens of 3 of 37 experts (21 get rows): 21 us, 2.2 TB/s, loads at odd addresses through registers
 *     fp32 2048 x 1024, 4 of 16 experts: 512 tokens 93 to 97 us, 89 to 93 TFLOP/s, one round of tiles, 27% of the matrix
 *     instructions on rows that are not there; 2048 tokens 244 us, 141; one token 28 us, 64 workgroups
 * The rows' gradient in tiles of 256 x 256 spills four registers, outside its loop.
 */
#include <hip/hip_runtime.h>
#include <type_traits>

#include "g53h.h"
#include "g53h_elem.h"
#include "g53h_mmtile.h"
#include "g53h_runtime.h"

#define G53_EM_MAXE 1024
#define G53_EM_MAXD (1 << 24)           /* rows and columns of a matrix */
#define G53_EM_MAXN (0x80000000l - 1024) /* pairs: chunks behind the last are counted in ints too */

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
    long wg0, wgs;                      /* first workgroup of the launch, workgroups of all      */
};

/* One tile of OP. DMA: operand rows start at multiples of 16 bytes and are whole pieces. */
template <typename E, int OP, int WR, int WC, int MT, int NT, int NS, bool DMA>
__global__ void __launch_bounds__(64 * WR * WC, MT * NT > 32 ? 1 : 2) k_emm(G53EmArgs a)
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
        const long item = g53_deal(wg, total);
        if (item >= total) return;
        it.e = (int)(item / per);
        int t;
        g53_eight(item % per, a.down, a.across, t, it.n);
        m0 = t * BM;
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

    /* Where a lane's pieces come from. Along: its row, and its place in 128 bytes. Across: its row of a chunk, whose places
     * repeat after VA or VB instructions; columns behind the last take the last piece (whole pieces) or what is there of
     * it: their results are not stored. */
    typedef G53Across<E, BM, MT> Xa;
    typedef G53Across<E, BN, NT> Xb;
    constexpr int KA = 64 / Xa::U, KB = 64 / Xb::U, VA = AX ? Xa::template turns<KA * NW>() : IA, VB = BX ? Xb::template turns<KB * NW>() : IB;
    const int u8 = (lane & 7) ^ (lane >> 3);
    const long wrow = (long)a.cols * sizeof(E), drow = (long)a.rows * sizeof(E);
    const uint8_t *pa[VA], *pb[VB];
    int ca[AX ? VA : 1], cb[BX ? VB : 1];                               /* across: first byte in a row */
#pragma unroll
    for (int i = 0; i < VA; i++) {
        if constexpr (!AX) {
            const int r = (i * NW + wv) * 8 + (lane >> 3), s = it.first + (r < live ? r : live - 1);
            pa[i] = OP == G53_EM_FWD ? a.x + token(s) * wrow + u8 * 16 : a.dy + s * drow + u8 * 16;
        } else {
            const int k = (i * NW + wv) * KA + lane / Xa::U;
            const long col = (long)m0 * sizeof(E) + ((lane % Xa::U) ^ Xa::place(k)) * 16;
            ca[i] = (int)(DMA && col > drow - 16 ? drow - 16 : col);
            pa[i] = a.dy + (it.first + k) * drow + ca[i];
        }
    }
#pragma unroll
    for (int i = 0; i < VB; i++) {
        if constexpr (!BX) {
            const int r = (i * NW + wv) * 8 + (lane >> 3);
            int at = n0 + r, up = 0;
            if (sw) {               /* a wave's first half of tiles: gate, the others: up */
                const int w = r / (16 * NT), t = r / 16 % NT;
                up = t >= NT / 2;
                at = n0 + w * (8 * NT) + (up ? t - NT / 2 : t) * 16 + r % 16;
            }
            at = at < a.half ? at : a.half - 1;
            pb[i] = we + (at + (up ? a.half : 0)) * wrow + u8 * 16;
        } else {
            const int k = (i * NW + wv) * KB + lane / Xb::U;
            const long col = (long)n0 * sizeof(E) + ((lane % Xb::U) ^ Xb::place(k)) * 16;
            cb[i] = (int)(DMA && col > wrow - 16 ? wrow - 16 : col);
            pb[i] = (OP == G53_EM_ROWS ? we + k * wrow : a.x) + cb[i];      /* matrices: the row joins it chunk by chunk */
        }
    }
    /* matrices: the tokens of an instruction's rows of x, asked for as scalars: their counter is not the loads' */
    int tok[OP == G53_EM_MATS ? IB : 1][KB];
    auto tokens = [&](int c) {
        if constexpr (OP == G53_EM_MATS)
#pragma unroll
            for (int i = 0; i < IB; i++)
#pragma unroll
                for (int r = 0; r < KB; r++) {
                    const int k = c * KE + (i * NW + wv) * KB + r, s = it.first + (k < live ? k : live - 1);
                    tok[i][r] = a.pair ? g53_uniform_load(a.pair + s) : s;
                }
    };
    const int kbytes = (int)(K * (long)sizeof(E));                      /* along: of a row */
    /* DMA: a row that is not there may have any address */
    auto piece_a = [&](int i, int c) -> G53Piece {
        if constexpr (!AX) {
            const uint8_t *p = pa[i];
            pa[i] += 128;
            return {p, kbytes - c * 128 - u8 * 16, true};
        } else {
            const int left = live - c * KE - (i * NW + wv) * KA, k = c * KE + i / VA * (VA * KA * NW);
            const bool row = lane / Xa::U < left;
            if constexpr (DMA) return {pa[i % VA] + k * drow, 16, row};
            return {pa[i % VA] + (row ? k : k + left - 1 - lane / Xa::U) * drow, (int)drow - ca[i % VA], row};
        }
    };
    auto piece_b = [&](int i, int c) -> G53Piece {
        if constexpr (!BX) {
            const uint8_t *p = pb[i];
            pb[i] += 128;
            return {p, kbytes - c * 128 - u8 * 16, true};
        } else {
            const int left = (int)K - c * KE - (i * NW + wv) * KB, n = DMA ? 16 : (int)wrow - cb[i % VB];
            const bool row = lane / Xb::U < left;
            if constexpr (OP == G53_EM_ROWS) {
                const uint8_t *p = pb[i % VB] + i / VB * (VB * KB * NW) * wrow;
                if (!DMA && !row) p += (left - 1 - lane / Xb::U) * wrow;
                if (i == IB - 1)
#pragma unroll
                    for (int v = 0; v < VB; v++) pb[v] += KE * wrow;
                return {p, n, row};
            }
            long t = 0;
#pragma unroll
            for (int r = 0; r < KB; r++) {
                const int pr = tok[OP == G53_EM_MATS ? i : 0][r];
                const long at = (long)(a.pair ? g53_div(pr, a.topk) : pr) * wrow;
                t = r == 0 || lane / Xb::U == r ? at : t;
            }
            return {pb[i % VB] + t, n, row};
        }
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    auto ask1 = [&](int c, int slot, int i) {               /* one instruction of a chunk */
        const G53Piece s = i < IA ? piece_a(i < IA ? i : 0, c) : piece_b(i < IA ? 0 : i - IA, c);
        const uint8_t *p = s.n > 0 && s.row ? s.p : (const uint8_t *)&g53_nothing;
        g53_to_lds(p, lds0 + slot * SLOT + wv * 1024 + (i < IA ? i * NW * 1024 : BM * 128 + (i - IA) * NW * 1024));
    };
    auto ask = [&](int c, int slot) {
        tokens(c);
#pragma unroll
        for (int i = 0; i < IA + IB; i++) ask1(c, slot, i);
    };
    /* small tiles: two sets, a chunk's pieces are asked for two chunks ahead (behind the last: somewhere in the rows) and put
     * down one ahead; large ones, whose registers would not hold them, one */
    constexpr int SETS = MT * NT <= 8 ? 2 : 1;
    g53_v4w ra[SETS][DMA ? 1 : IA], rb[SETS][DMA ? 1 : IB];
    int bya[SETS][DMA ? 1 : IA], byb[SETS][DMA ? 1 : IB];
    const bool short_a = (AX ? drow : kbytes) < 16, short_b = (BX ? wrow : kbytes) < 16;
    auto fetch = [&](int c, int set) {
        if constexpr (!DMA) {
            tokens(c);
            if (short_a || short_b) {
#pragma unroll
                for (int i = 0; i < IA; i++) g53_take_short<E>(ra[set][i], bya[set][i], piece_a(i, c));
#pragma unroll
                for (int i = 0; i < IB; i++) g53_take_short<E>(rb[set][i], byb[set][i], piece_b(i, c));
            } else {
#pragma unroll
                for (int i = 0; i < IA; i++) g53_take(ra[set][i], bya[set][i], piece_a(i, c));
#pragma unroll
                for (int i = 0; i < IB; i++) g53_take(rb[set][i], byb[set][i], piece_b(i, c));
            }
        }
    };
    auto put = [&](int slot, int set) {
        if constexpr (!DMA) {
            uint8_t *to = lds + slot * SLOT + wv * 1024 + lane * 16;
#pragma unroll
            for (int i = 0; i < IA; i++) *(g53_v4w *)(to + i * NW * 1024) = g53_moved<E>(ra[set][i], bya[set][i]);
#pragma unroll
            for (int i = 0; i < IB; i++) *(g53_v4w *)(to + BM * 128 + i * NW * 1024) = g53_moved<E>(rb[set][i], byb[set][i]);
        }
    };

    typename std::conditional<AX, G53Across<E, BM, MT, WR>, G53Along<E, WR>>::type fa;
    typename std::conditional<BX, G53Across<E, BN, NT>, G53Along<E>>::type fb;
    fa.setup(wr * 16);                  /* tile i of wave row wr is the tile's 16 rows i * WR + wr: rows that are there spread over all */
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
    if constexpr (DMA && STEPS == 2) {
        /* Operands of one step are in registers while those of the next leave LDS between its products. The slot of chunk c
         * is free once its second step's operands are read, halfway through the chunk: there one barrier hands it to chunk
         * c + NS, and says that c + 1 is there, whose first step's operands are read beside the second half's products. */
        auto run = [&](auto M_) {
        constexpr int M = decltype(M_)::value;                  /* row tiles of a wave that are there */
        G53Frag<E> va[2][M], vb[2][NT];
        auto read1 = [&](int to, int slot, int j, int i) {  /* one fragment of a step */
            const uint8_t *la = lds + slot * SLOT;
            if (i < NT) fb.read(vb[to][i], la + BM * 128, i, j);
            else fa.read(va[to][i - NT], la, i - NT, j);
        };
        constexpr int RD = (M + NT + M - 1) / M, IM = AX ? IA : IA * M / MT, AD = (IM + IB + M - 1) / M;
        if (chunks) {
#pragma unroll
            for (int c = 0; c < NS; c++) {
                tokens(c);
#pragma unroll
                for (int i = 0; i < IM + IB; i++) ask1(c, c, i < IM ? i : i - IM + IA);
            }         /* behind the last chunk: zeros, which nothing uses */
            g53_loads_left<(NS - 1) * (IM + IB)>();
            g53_meet();
#pragma unroll
            for (int i = 0; i < M + NT; i++) read1(0, 0, 0, i);
        }
        int slot = 0;
        for (int c = 0; c < chunks; c++) {
            tokens(c + NS);
#pragma unroll
            for (int i = 0; i < M; i++) {
#pragma unroll
                for (int k = i * RD; k < (i + 1) * RD && k < M + NT; k++) read1(1, slot, 1, k);
#pragma unroll
                for (int t = 0; t < NT; t++) acc[i][t] = g53_mm<E>(vb[0][t], va[0][i], acc[i][t]);
                __builtin_amdgcn_sched_barrier(0);
            }
            g53_loads_left<(NS - 2) * (IM + IB)>();
            g53_meet();
            const int next = slot == NS - 1 ? 0 : slot + 1;
#pragma unroll
            for (int i = 0; i < M; i++) {
#pragma unroll
                for (int k = i * AD; k < (i + 1) * AD && k < IM + IB; k++) ask1(c + NS, slot, k < IM ? k : k - IM + IA);
#pragma unroll
                for (int k = i * RD; k < (i + 1) * RD && k < M + NT; k++) read1(0, next, 0, k);
#pragma unroll
                for (int t = 0; t < NT; t++) acc[i][t] = g53_mm<E>(vb[1][t], va[1][i], acc[i][t]);
                __builtin_amdgcn_sched_barrier(0);
            }
            slot = next;
        }
        g53_loads_left<0>();                                /* no load outlives the workgroup's LDS */
        };
        typedef std::integral_constant<int, MT> All;
        if constexpr (AX || MT < 8) run(All{});
        else if (live <= BM / 4) run(std::integral_constant<int, MT / 4>{});
        else if (live <= BM / 2) run(std::integral_constant<int, MT / 2>{});
        else run(All{});
    } else if constexpr (DMA) {
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
            fetch(0, 0);
            if (SETS == 2) fetch(1, SETS - 1);
            put(0, 0);
        }
        if constexpr (SETS == 2) {
            for (int c = 0; c < chunks; c += 2) {
                __syncthreads();
                fetch(c + 2, 0);
                multiply(0);
                put(1, SETS - 1);
                if (c + 1 >= chunks) break;
                __syncthreads();
                fetch(c + 3, SETS - 1);
                multiply(1);
                put(0, 0);
            }
        } else {
            for (int c = 0; c < chunks; c++) {
                __syncthreads();
                fetch(c + 1, 0);
                multiply(c & 1);
                put(c + 1 & 1, 0);
            }
        }
    }

    /* out: the loads' slots hold the wave's tiles on their way */
    g53_meet();
    if constexpr (OP == G53_EM_MATS) {
        const int r0 = m0 + wr * 16, c0 = n0 + wc * NT * 16;
        static_assert(NS * SLOT >= NW * MT * NT * 1024, "tiles on their way out");
        g53_leave_sums<E, WR>(lds + wv * (MT * NT * 1024), a.out, ((long)it.e * a.rows + r0) * a.cols + c0, a.cols, acc, a.rows - r0,
                              a.cols - c0, a.w_f32, a.add);
    } else {
        static_assert(NS * SLOT >= NW * MT * NT * 256 * (int)sizeof(E), "tiles on their way out");
        uint8_t *const buf = lds + wv * (MT * NT * 256 * (int)sizeof(E));
        const int r0 = wr * 16, N = OP == G53_EM_ROWS ? a.cols : a.half;
        const long first = it.first + r0;
        if constexpr (OP == G53_EM_FWD)
            if (sw) {
                const int c = n0 + wc * (NT / 2 * 16), most = a.half - c;
                g53_v4f v[MT][NT / 2];
                if (a.gu) {                                     /* gate, then up: the rows' second halves */
                    E *at = (E *)a.gu + first * a.rows + c;
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int t = 0; t < NT / 2; t++) v[i][t] = acc[i][t];
                    g53_leave<E, WR>(buf, at, a.rows, v, live - r0, most);
#pragma unroll
                    for (int i = 0; i < MT; i++)
#pragma unroll
                        for (int t = 0; t < NT / 2; t++) v[i][t] = acc[i][t + NT / 2];
                    g53_leave<E, WR>(buf, at + a.half, a.rows, v, live - r0, most);
                }
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int t = 0; t < NT / 2; t++)
#pragma unroll
                        for (int k = 0; k < 4; k++) v[i][t][k] = g53_swiglu1<E>(acc[i][t][k], acc[i][t + NT / 2][k], a.limit);
                g53_leave<E, WR>(buf, (E *)a.out + first * N + c, N, v, live - r0, most);
                return;
            }
        const int c = n0 + wc * NT * 16;
        g53_leave<E, WR>(buf, (E *)a.out + first * N + c, N, acc, live - r0, N - c);
    }
}

/* The matrices' gradient in 16 bits, of whole pieces. An expert's rows are few next to a matrix (a tile of results often
 * takes less time to sum than to write), so workgroups stay and go from tile to tile: while a tile's last chunks are
 * multiplied and its results leave, the next one's first chunks are on their way. The stream of chunks passes experts
 * without rows, whose tiles are zeros. */
template <typename E, int WR, int WC, int MT, int NT, int NS>
__global__ void __launch_bounds__(64 * WR * WC, MT * NT > 32 ? 1 : 2) k_emats(G53EmArgs a)
{
    constexpr int NW = WR * WC, BM = 16 * MT * WR, BN = 16 * NT * WC, SLOT = (BM + BN) * 128, KE = 64;
    constexpr int IA = BM / (8 * NW), IB = BN / (8 * NW);
    typedef G53Across<E, BM, MT> Xa;
    typedef G53Across<E, BN, NT> Xb;
    constexpr int KA = 64 / Xa::U, KB = 64 / Xb::U;                     /* rows of a wave's instruction */
    constexpr int VA = Xa::template turns<KA * NW>(), VB = Xb::template turns<KB * NW>();    /* after as many, places repeat */
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wv / WC, wc = wv % WC;
    const long wrow = (long)a.cols * sizeof(E), drow = (long)a.rows * sizeof(E);
    const int per = a.across * a.down;
    /* tiles: fewer than 2^31 (each has 128 elements of memory and more, or is an expert's only one) */
    const unsigned total = (unsigned)a.NE * per;
    /* the tile of a workgroup's turn w: runs of tiles by die, eight tiles down with each across */
    struct Tile {
        int e, m0, n0, first, live;
    };
    auto tile_of = [&](unsigned w, Tile &t) {
        const unsigned item = g53_deal(w, total);
        if (item >= total) return false;
        t.e = (int)(item / per);
        int m, n;
        g53_eight(item - (unsigned)t.e * per, a.down, a.across, m, n);
        t.m0 = m * BM;
        t.n0 = n * BN;
        t.first = g53_uniform_load(a.offsets + t.e);
        t.live = g53_uniform_load(a.offsets + t.e + 1) - t.first;
        return true;
    };
    const unsigned turns = (unsigned)a.wgs;
    /* The stream: the tile and chunk to be asked for (none behind the last: zeros), and the one after it, whose tokens
     * are asked for a chunk ahead. */
    struct At {
        Tile t;
        int c, chunks, left;            /* left: rows from the chunk's first on, 0 behind the last tile */
    };
    At s, nx;
    unsigned nw = blockIdx.x;
    auto seek = [&]() {
        nx.c = nx.chunks = 0;
        for (; nw < turns; nw += gridDim.x)
            if (tile_of(nw, nx.t) && nx.t.live) {
                nx.chunks = (nx.t.live + KE - 1) / KE;
                break;
            }
    };
    const uint8_t *pa[VA];
    int cb[VB], tok[IB], tokn[IB];
    const int ka = wv * KA + lane / Xa::U, kb = wv * KB + lane / Xb::U;
    auto tokens = [&]() {
        if (!nx.chunks) return;
#pragma unroll
        for (int i = 0; i < IB; i++) {
            const int k = nx.c * KE + kb + i * KB * NW, r = nx.t.first + (k < nx.t.live ? k : nx.t.live - 1);
            tokn[i] = a.pair ? a.pair[r] : r;
        }
    };
    auto on = [&]() {                                       /* to the stream's next chunk */
        s = nx;
        s.left = s.chunks ? s.t.live - s.c * KE : 0;
#pragma unroll
        for (int i = 0; i < IB; i++) tok[i] = tokn[i];
        if (!s.chunks) return;
        if (!s.c) {
#pragma unroll
            for (int v = 0; v < VA; v++) {
                const int k = ka + v * KA * NW;
                long col = (long)s.t.m0 * sizeof(E) + ((lane % Xa::U) ^ Xa::place(k)) * 16;
                col = col > drow - 16 ? drow - 16 : col;    /* columns behind the last: not stored */
                pa[v] = a.dy + (long)(s.t.first + k) * drow + col;
            }
#pragma unroll
            for (int v = 0; v < VB; v++) {
                const long col = (long)s.t.n0 * sizeof(E) + ((lane % Xb::U) ^ Xb::place(kb + v * KB * NW)) * 16;
                cb[v] = (int)(col > wrow - 16 ? wrow - 16 : col);
            }
        } else {
#pragma unroll
            for (int v = 0; v < VA; v++) pa[v] += KE * drow;
        }
        if (++nx.c == nx.chunks) {
            nw += gridDim.x;
            seek();
        }
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    auto ask1 = [&](int slot, int i) {                      /* one instruction of the stream's chunk */
        const uint32_t to = lds0 + slot * SLOT + wv * 1024;
        const uint8_t *p = (const uint8_t *)&g53_nothing;
        if (i < IA) {
            const uint8_t *at = pa[i % VA] + (i / VA) * (VA * KA * NW) * drow;
            p = lane / Xa::U < s.left - (i * NW + wv) * KA ? at : p;
            g53_to_lds(p, to + i * NW * 1024);
        } else {
            const int j = i - IA;
            const uint8_t *at = a.x + (long)g53_div(tok[j], a.topk) * wrow + cb[j % VB];
            p = lane / Xb::U < s.left - (j * NW + wv) * KB ? at : p;
            g53_to_lds(p, to + BM * 128 + j * NW * 1024);
        }
    };
    Xa fa;
    Xb fb;
    fa.setup(wr * 16 * MT);
    fb.setup(wc * 16 * NT);
    G53Frag<E> va[2][MT], vb[2][NT];
    auto read1 = [&](int to, int slot, int j, int i) {      /* one fragment of a step */
        const uint8_t *l = lds + slot * SLOT;
        if (i < NT) fb.read(vb[to][i], l + BM * 128, i, j);
        else fa.read(va[to][i - NT], l, i - NT, j);
    };
    constexpr int RD = (MT + NT + MT - 1) / MT, AD = 2 * ((IA + IB + MT - 1) / MT);
    seek();
    tokens();
    on();
#pragma unroll
    for (int c = 0; c < NS; c++) {
        tokens();
#pragma unroll
        for (int i = 0; i < IA + IB; i++) ask1(c, i);
        on();
    }
    g53_loads_left<(NS - 1) * (IA + IB)>();
    g53_meet();
#pragma unroll
    for (int i = 0; i < MT + NT; i++) read1(0, 0, 0, i);
    int slot = 0;
    for (unsigned w = blockIdx.x; w < turns; w += gridDim.x) {
        Tile t;
        if (!tile_of(w, t) || (a.add && !t.live)) continue;
        g53_v4f acc[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = (g53_v4f){0.0f, 0.0f, 0.0f, 0.0f};
        const int chunks = (t.live + KE - 1) / KE;
        for (int c = 0; c < chunks; c++) {                  /* see k_emm */
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int k = i * RD; k < (i + 1) * RD && k < MT + NT; k++) read1(1, slot, 1, k);
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] = g53_mm<E>(vb[0][j], va[0][i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            g53_loads_left<(NS - 2) * (IA + IB)>();
            g53_meet();
            const int next = slot == NS - 1 ? 0 : slot + 1;
            tokens();
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int k = i * AD; k < (i + 1) * AD && k < IA + IB; k++) ask1(slot, k);
#pragma unroll
                for (int k = i * RD; k < (i + 1) * RD && k < MT + NT; k++) read1(0, next, 0, k);
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] = g53_mm<E>(vb[1][j], va[1][i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            slot = next;
            on();
        }
        const int r0 = t.m0 + wr * 16 * MT, c0 = t.n0 + wc * 16 * NT;
        uint8_t *const buf = lds + NS * SLOT + wv * (NT * 1024);
#pragma unroll
        for (int i = 0; i < MT; i++) {                      /* LDS beside the slots holds a row of tiles */
            const int r = r0 + 16 * i;
            g53_v4f v[1][NT];
#pragma unroll
            for (int j = 0; j < NT; j++) v[0][j] = acc[i][j];
            g53_leave_sums<E, 1>(buf, a.out, ((long)t.e * a.rows + r) * a.cols + c0, a.cols, v, a.rows - r, a.cols - c0, a.w_f32, a.add);
        }
    }
    g53_loads_left<0>();                                    /* no load outlives the workgroup's LDS */
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
    const long wgs = g53_deal_wgs(items);
    for (long w0 = 0; w0 < wgs; w0 += G53_EM_WGS) {
        a.wg0 = w0;
        const dim3 grid((unsigned)(wgs - w0 < G53_EM_WGS ? wgs - w0 : G53_EM_WGS));
        hipLaunchKernelGGL((k_emm<E, OP, WR, WC, MT, NT, NS, DMA>), grid, dim3(64 * WR * WC), LDS, g53h_stream(), a);
        G53_LAUNCHED("k_emm");
    }
    return 0;
}

template <typename E, int WR, int WC, int MT, int NT, int NS> static int matrices(G53EmArgs a)
{
    constexpr int BM = 16 * MT * WR, BN = 16 * NT * WC;
    constexpr size_t LDS = (size_t)NS * (BM + BN) * 128 + WR * WC * NT * 1024;
    static int allowed = 0;
    if (!allowed) {
        G53_TRY(hipFuncSetAttribute((const void *)k_emats<E, WR, WC, MT, NT, NS>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)LDS));
        allowed = 1;
    }
    a.across = (a.cols + BN - 1) / BN;
    a.down = (a.rows + BM - 1) / BM;
    const long total = (long)a.NE * a.down * a.across, stay = g53h_num_cus() / 8 * 8 * (LDS > 80 * 1024 ? 1 : 2);
    a.wgs = g53_deal_wgs(total);
    const dim3 grid((unsigned)(a.wgs < stay ? a.wgs : stay));
    hipLaunchKernelGGL((k_emats<E, WR, WC, MT, NT, NS>), grid, dim3(64 * WR * WC), LDS, g53h_stream(), a);
    G53_LAUNCHED("k_emats");
    return 0;
}

template <typename E, int OP> static int by_size(const G53EmArgs &a, long n)
{
    /* whole pieces of 16 bytes at multiples of 16 */
    const uintptr_t at = OP == G53_EM_FWD ? (uintptr_t)a.x | (uintptr_t)a.w
                         : OP == G53_EM_ROWS ? (uintptr_t)a.dy | (uintptr_t)a.w : (uintptr_t)a.dy | (uintptr_t)a.x;
    const size_t odd = (a.cols * sizeof(E)) | (OP == G53_EM_FWD ? 0 : a.rows * sizeof(E));
    /* Few rows an expert, or few tiles of the matrices: tiles of 32 x 128, of which more are at work at a time. us, 2048 x 1024,
     * 16 experts, top-4, 1, 32, 256 and 2048 tokens, tiles of 128 x 128 / 32 x 128: forward fp32 56 59 70 240 / 28 34 59 299,
     * fp16 of 1023 columns 26 31 34 101 / 18 20 31 147; rows fp32 110 111 112 276 / 55 56 76 296; matrices fp32 57 50 58 228 /
     * 43 34 64 313. The tests repeat the rules below, to name the tile that a size takes. */
    const long busy = a.NE < n ? a.NE : n, mean = busy ? (n + busy - 1) / busy : 0, cus = g53h_num_cus();
    const bool few = OP == G53_EM_MATS ? (long)a.NE * ((a.rows + 127) / 128) * ((a.cols + 127) / 128) < cus : mean <= 64;
    if constexpr (OP == G53_EM_ROWS) {      /* fewer still: a wave's part of a chunk is what takes time */
        if (few && (n / 32 + busy) * ((a.cols + 127) / 128) < cus) {
            if ((at | odd) & 15) return launch<E, OP, 1, 4, 2, 1, 2, false>(a, n);
            if constexpr (sizeof(E) == 4) return launch<E, OP, 1, 4, 2, 1, 4, true>(a, n);
        }
    }
    if ((at | odd) & 15) return few ? launch<E, OP, 1, 4, 2, 2, 2, false>(a, n) : launch<E, OP, 2, 2, 4, 4, 2, false>(a, n);
    if constexpr (sizeof(E) == 4) {
        return few ? launch<E, OP, 1, 4, 2, 2, 4, true>(a, n) : launch<E, OP, 2, 2, 4, 4, 2, true>(a, n);
    } else if constexpr (OP == G53_EM_MATS) {
        return matrices<E, 2, 2, 4, 4, 2>(a);
    } else {
        /* Experts' rows count as all alike, since the host does not know them. Tiles of 256 x 256 read LDS least for a
         * product, where there are as many as CUs; of 128 x 128 where there are two a CU; few rows take tiles of 64 x 128 and
         * 32 x 128, of which two workgroups a CU keep up to 96 KB of matrices on their way. us, bf16, forward / rows:
         *     4096 x 4096, 64 experts, top-8   256       128       64 x 256  64 x 128  32 x 128
         *     4096 tokens                  1094/1269 1299/1319 1534/1522 1601/1581 2286/2259
         *     1024                           423/476   465/469   507/480   518/505   723/697
         *     256                            307/265   296/267   295/247   284/263   319/291
         *     1                               74/78     66/66     55/53     50/48     49/48
         *     2048 x 1024, 32 experts, top-4
         *     1024                            39/67     46/43     49/54     48/47     60/59
         *     64                              23/40     21/32     18/26     19/19     18/19                              */
        const int N = OP == G53_EM_FWD ? a.rows : a.cols;
        auto tiles = [&](int bm, int bn) { return (n / bm + busy) * ((N + bn - 1) / bn); };
        if (mean >= 64 && tiles(256, 256) >= cus) return launch<E, OP, 2, 2, 8, 8, 2, true>(a, n);
        if (mean >= 128 && tiles(128, 128) >= 2 * cus) return launch<E, OP, 2, 2, 4, 4, 2, true>(a, n);
        if (OP == G53_EM_ROWS && mean > 1 && tiles(64, 256) >= 2 * cus) return launch<E, G53_EM_ROWS, 1, 4, 4, 4, 3, true>(a, n);
        if (mean > 4 && tiles(64, 128) >= 2 * cus) return launch<E, OP, 1, 4, 4, 2, 3, true>(a, n);
        return launch<E, OP, 1, 4, 2, 2, 3, true>(a, n);
    }
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
        /* below -1000, where the sigmoid is 0, any gate is -1000: with the 0, -inf (as a gate past fp16 is kept) and what
         * overflows next to the type's lowest value would give NaN */
        const float gc = g[i] > limit ? limit : (g[i] < -1000.0f ? -1000.0f : g[i]);
        const float uc = u[i] > limit ? limit : (u[i] < -limit ? -limit : u[i]);
        const bool low = gc < -80.0f;       /* there 1 + exp(g) is 1, and exp(-g) may overflow */
        const float x = expf(low ? gc : -gc), s = low ? x : 1.0f / (1.0f + x);
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
        (long)p->T * p->topk > G53_EM_MAXN || !p->offsets || (p->T && !p->pair))
        return g53h_fail("%s: no plan of g53h_sort_tokens (of at most 2^31 - 1024 pairs)", who);
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
        if (!gather) a.topk = g53_div_of(1);
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
