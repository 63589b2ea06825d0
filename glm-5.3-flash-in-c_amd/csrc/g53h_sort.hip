/* g53h_sort.hip - tokens sorted by expert and back: the order of a routing's (token, slot) pairs by
 * expert (a stable counting sort), the copy of every token's row to its experts' rows, the weighted
 * sum back, and the gradients of both.
 *
 * k_sort_place: a pair's row is offsets[its expert] + the number of earlier pairs of the same expert. A
 * workgroup counts its pairs per wave and expert in LDS, turns the counts into first rows by a prefix sum
 * over the experts and the waves, and then walks its pairs in order, 64 at a time: a ballot per bit of the
 * expert gives each lane the lanes with the same expert, those below it are its rank. Order never depends on
 * timing. Routings of more than G53_SORT_SEG pairs are cut into segments, counted by k_sort_count first;
 * every workgroup then adds up the counts of all segments. Latency: 2.6 us for 64 pairs and fewer
 * (k_sort_few), 4.8 + 7.8 for 32768 pairs of 288 experts in 16 segments (9.7 in a row of sorts).
 *
 * k_sorted_dispatch: bytes of rows, 16 a thread; a token's row is read once and written topk times. 4096
 * tokens of 4096 bf16 to 8 experts each, 302 MB: 55 us, 5.5 TB/s, bound by HBM. Written past the caches the
 * rows alone leave faster (with the sort and a combine of other rows after it 128 us against 136), but
 * whoever reads them next waits longer (dispatch and a read of its rows 104 us against 93; 67 MB of rows 28
 * against 25).
 *
 * k_sorted_combine: 8 elements a thread; the rows of a token's pairs are all asked for before the first is
 * added; sums in fp32 in the order of the pairs, rounded once. The same tokens, 302 MB: 68 us, 4.4 TB/s, a
 * large copy's rate.
 *
 * k_sorted_combine_grad: one wave per pair. Its weight's gradient is one sum over the wave, so nothing is
 * exchanged between waves; the waves of a workgroup mostly share a token, whose gradient row they read from
 * the vector cache. 2048 of these tokens, 285 MB: 64 us, 4.5 TB/s.
 */
#include <hip/hip_runtime.h>

#include "g53h.h"
#include "g53h_elem.h"
#include "g53h_runtime.h"

#define G53_SORT_SEG 2048               /* pairs of one workgroup, while there are at most G53_SORT_WGS */
#define G53_SORT_WGS 128
#define G53_SORT_MAXE 1024

/* ------------------------------------------------------------------------- sort ---- */
/* Pairs [first, last) of a launch's segment `seg`. */
__device__ __forceinline__ void g53_seg(long n, int per, int seg, long &first, long &last)
{
    first = (long)seg * per;
    last = first + per < n ? first + per : n;
}

__global__ void __launch_bounds__(1024) k_sort_count(int *__restrict__ hist, const int *__restrict__ idx, long n, int per,
                                                     int NE)
{
    __shared__ int cnt[G53_SORT_MAXE];
    for (int e = threadIdx.x; e < NE; e += 1024) cnt[e] = 0;
    __syncthreads();
    long first, last;
    g53_seg(n, per, blockIdx.x, first, last);
    for (long i = first + threadIdx.x; i < last; i += 1024) {
        const int e = idx[i];
        if ((unsigned)e < (unsigned)NE) atomicAdd(&cnt[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < NE; e += 1024) hist[(long)blockIdx.x * NE + e] = cnt[e];
}

/* hist: counts [gridDim.x][NE] of all segments (unused where there is one). NW waves a workgroup;
 * first [NW][NE] in dynamic LDS. bits: of the largest expert. */
template <int NW>
__global__ void __launch_bounds__(64 * NW)
k_sort_place(int *__restrict__ offsets, int *__restrict__ pair, int *__restrict__ row, const int *__restrict__ idx,
             const int *__restrict__ hist, long n, int per, int NE, int bits)
{
    extern __shared__ int first_of[];   /* [NW][NE]: pairs of a wave, then the next row of its expert */
    __shared__ int wsum[NW];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    for (int i = tid; i < NW * NE; i += 64 * NW) first_of[i] = 0;
    __syncthreads();
    long s0, s1;
    g53_seg(n, per, blockIdx.x, s0, s1);
    /* whole steps of 64 pairs a wave */
    const long wper = ((s1 - s0 + 64 * NW - 1) / (64 * NW)) * 64;
    const long w0 = s0 + wv * wper, w1 = w0 + wper < s1 ? w0 + wper : s1;
    int *mine = first_of + wv * NE;
    for (long i = w0 + lane; i < w1; i += 64) {
        const int e = idx[i];
        if ((unsigned)e < (unsigned)NE) atomicAdd(&mine[e], 1);
    }
    __syncthreads();
    int base = 0;                       /* pairs of all experts before this round's */
    for (int e0 = 0; e0 < NE; e0 += 64 * NW) {
        const int e = e0 + tid;
        int total = 0, before = 0, here = 0;
        if (e < NE) {
            for (int w = 0; w < NW; w++) here += first_of[w * NE + e];
            if (gridDim.x == 1) total = here;
            else
#pragma unroll 16
                for (int b = 0; b < (int)gridDim.x; b++) {      /* loads of 16 segments in flight */
                    const int c = hist[(long)b * NE + e];
                    total += c;
                    before += b < (int)blockIdx.x ? c : 0;
                }
        }
        int incl = total;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        if (lane == 63) wsum[wv] = incl;
        __syncthreads();
        int start = base + incl - total;
        for (int w = 0; w < NW; w++) {
            start += w < wv ? wsum[w] : 0;
            base += wsum[w];
        }
        if (e < NE) {
            if (blockIdx.x == 0) offsets[e] = start;
            int at = start + before;
            for (int w = 0; w < NW; w++) {
                const int c = first_of[w * NE + e];
                first_of[w * NE + e] = at;
                at += c;
            }
        }
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) offsets[NE] = base;
    for (long i0 = w0; i0 < w1; i0 += 64) {
        const long i = i0 + lane;
        const int e = i < w1 ? idx[i] : -1;
        const bool in = (unsigned)e < (unsigned)NE;
        unsigned long long same = __ballot(in);
        for (int b = 0; b < bits; b++) {
            const unsigned long long set = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? set : ~set;
        }
        int at = -1;
        if (in) {
            at = mine[e] + __popcll(same & ((1ull << lane) - 1));
            pair[at] = (int)i;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");   /* the lanes' reads before the update */
        __builtin_amdgcn_wave_barrier();
        if (in && (same >> lane) == 1ull) mine[e] = at + 1;      /* the last lane of its expert */
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (i < w1) row[i] = at;
    }
    for (long p = base + (long)blockIdx.x * (64 * NW) + tid; p < n; p += (long)gridDim.x * (64 * NW)) pair[p] = -1;
}

/* Up to 64 pairs: a lane holds a pair's key and meets every other; experts count the keys below them. No LDS, no barrier:
 * one token's 8 pairs of 288 experts in 2.6 us, a launch's own time, against 4.1 by counting. */
__global__ void __launch_bounds__(256) k_sort_few(int *__restrict__ offsets, int *__restrict__ pair, int *__restrict__ row,
                                                  const int *__restrict__ idx, int n, int NE)
{
    const int tid = threadIdx.x, lane = tid & 63;
    int key = NE;                       /* left out, or no pair: behind every expert */
    if (lane < n) {
        const int e = idx[lane];
        if ((unsigned)e < (unsigned)NE) key = e;
    }
    const int total = __popcll(__ballot(key < NE));
    for (int e0 = 0; e0 <= NE; e0 += 256) {
        const int e = e0 + tid;
        int below = 0;
        for (int j = 0; j < n; j++) below += __builtin_amdgcn_readlane(key, j) < e;
        if (e <= NE) offsets[e] = below;
    }
    if (tid >= 64) return;
    int at = 0;
    for (int j = 0; j < n; j++) {
        const int k = __builtin_amdgcn_readlane(key, j);
        at += k < key || (k == key && j < lane);
    }
    if (lane >= n) return;
    row[lane] = key < NE ? at : -1;
    if (key < NE) pair[at] = lane;
    if (lane >= total) pair[lane] = -1;
}

/* A routing's plan: sizes that fit, arrays that are there. */
static int sort_bad(const G53hSort *p, const char *who)
{
    if (!p) return g53h_fail("%s: no plan", who);
    if (p->T < 0 || p->topk < 1 || p->topk > 64 || p->n_experts < 1 || p->n_experts > G53_SORT_MAXE ||
        (long)p->T * p->topk > 0x7fffffffl)
        return g53h_fail("%s: %d tokens of %d experts out of %d (topk 1 to 64, at most %d experts, pairs below 2^31)", who,
                         p->T, p->topk, p->n_experts, G53_SORT_MAXE);
    if (!p->offsets || (p->T && (!p->pair || !p->row))) return g53h_fail("%s: plan without its arrays", who);
    return 0;
}

extern "C" int g53h_sort_tokens(const G53hSort *p, const int *idx)
{
    if (sort_bad(p, "g53h_sort_tokens")) return -1;
    if (p->T && !idx) return g53h_fail("g53h_sort_tokens: no routing");
    if (g53h_ready()) return -1;
    const long n = (long)p->T * p->topk;
    const int NE = p->n_experts;
    if (n <= 64) {
        hipLaunchKernelGGL(k_sort_few, dim3(1), dim3(256), 0, g53h_stream(), p->offsets, p->pair, p->row, idx, (int)n, NE);
        G53_LAUNCHED("k_sort_few");
        return 0;
    }
    int bits = 0;
    while ((1 << bits) < NE) bits++;
    long wgs = (n + G53_SORT_SEG - 1) / G53_SORT_SEG;
    wgs = wgs < 1 ? 1 : (wgs > G53_SORT_WGS ? G53_SORT_WGS : wgs);
    const int per = (int)((n + wgs - 1) / wgs);
    int *hist = nullptr;
    static int allowed = 0;             /* 1024 experts: 64 KB of counts and a little more */
    if (!allowed) {
        G53_TRY(hipFuncSetAttribute((const void *)k_sort_place<16>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                    16 * G53_SORT_MAXE * 4));
        allowed = 1;
    }
    if (wgs > 1) {
        hist = (int *)g53h_op_workspace((size_t)wgs * NE * sizeof(int));
        if (!hist) return -1;
        hipLaunchKernelGGL(k_sort_count, dim3((unsigned)wgs), dim3(1024), 0, g53h_stream(), hist, idx, n, per, NE);
        G53_LAUNCHED("k_sort_count");
    }
    if (n <= 1024)
        hipLaunchKernelGGL(k_sort_place<4>, dim3(1), dim3(256), 4 * NE * sizeof(int), g53h_stream(), p->offsets, p->pair,
                           p->row, idx, hist, n, per, NE, bits);
    else
        hipLaunchKernelGGL(k_sort_place<16>, dim3((unsigned)wgs), dim3(1024), 16 * NE * sizeof(int), g53h_stream(),
                           p->offsets, p->pair, p->row, idx, hist, n, per, NE, bits);
    G53_LAUNCHED("k_sort_place");
    return 0;
}

/* --------------------------------------------------------------------- dispatch ---- */
/* nb bytes a row; a workgroup copies 4 KB of one token's row to its topk rows. */
__global__ void __launch_bounds__(256) k_sorted_dispatch(uint8_t *__restrict__ xs, const uint8_t *__restrict__ x,
                                                  const int *__restrict__ row, long nb, int K, int chunks, long wg0)
{
    const long wg = wg0 + blockIdx.x;
    const long t = wg / chunks, at = ((wg % chunks) * 256 + threadIdx.x) * 16;
    if (at >= nb) return;
    const uint8_t *src = x + t * nb + at;
    const int *r = row + t * K;
    if (at + 16 <= nb) {
        const g53_v4w v = ((const G53v4w_any *)src)->v;
        for (int j = 0; j < K; j++)
            if (r[j] >= 0) ((G53v4w_any *)(xs + r[j] * nb + at))->v = v;
    } else {
        for (int j = 0; j < K; j++)
            if (r[j] >= 0)
                for (int i = 0; at + i < nb; i += 2) *(uint16_t *)(xs + r[j] * nb + at + i) = *(const uint16_t *)(src + i);
    }
}

/* Workgroups that one launch takes: its threads, and those of every launch here are at most 256 a
 * workgroup, are counted in 32 bits. */
#define G53_LAUNCH_WGS (1l << 23)

static int rows_bad(const char *who, const G53hSort *p, int dt, int hidden)
{
    if (sort_bad(p, who)) return -1;
    if (!g53_elem_bytes(dt)) return g53h_fail("%s: element type %d", who, dt);
    if (hidden < 1 || hidden > 1 << 30) return g53h_fail("%s: hidden %d", who, hidden);
    return 0;
}

extern "C" int g53h_sorted_dispatch(void *xs, const void *x, int dt, int hidden, const G53hSort *p)
{
    if (rows_bad("g53h_sorted_dispatch", p, dt, hidden)) return -1;
    if (!p->T) return 0;
    if (!xs || !x) return g53h_fail("g53h_sorted_dispatch: no rows");
    if (g53h_ready()) return -1;
    const long nb = (long)hidden * g53_elem_bytes(dt);
    const int chunks = (int)((nb + 4095) / 4096);
    const long total = (long)p->T * chunks;
    for (long w0 = 0; w0 < total; w0 += G53_LAUNCH_WGS) {
        const unsigned wgs = (unsigned)(total - w0 < G53_LAUNCH_WGS ? total - w0 : G53_LAUNCH_WGS);
        hipLaunchKernelGGL(k_sorted_dispatch, dim3(wgs), dim3(256), 0, g53h_stream(), (uint8_t *)xs, (const uint8_t *)x, p->row, nb,
                           p->topk, chunks, w0);
        G53_LAUNCHED("k_sorted_dispatch");
    }
    return 0;
}

/* ---------------------------------------------------------------------- combine ---- */
/* out[t] = add[t] + sum over the token's pairs of w times their row; w NULL: 1, add NULL: 0. */
template <typename E>
__global__ void __launch_bounds__(256) k_sorted_combine(E *out, const E *__restrict__ ys, const float *__restrict__ w,
                                                 const E *add, const int *__restrict__ row, int H, int K, int chunks,
                                                 long wg0)
{
    const long wg = wg0 + blockIdx.x;
    const long t = wg / chunks;
    const int c = ((int)(wg % chunks) * 256 + threadIdx.x) * 8;
    if (c >= H) return;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (add) g53_load8_to(acc, add + t * H, c, H);
    for (int j0 = 0; j0 < K; j0 += 8) {
        G53Raw8<E> v[8];
        int r[8];
        float wj[8];                    /* asked for with the rows' places, not behind the rows */
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const long at = t * K + (j0 + j < K ? j0 + j : K - 1);
            r[j] = j0 + j < K ? row[at] : -1;
            wj[j] = w ? w[at] : 1.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (r[j] >= 0) g53_raw8_once_to(v[j], ys + (long)r[j] * H, c, H);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (r[j] >= 0)
#pragma unroll
                for (int i = 0; i < 8; i++) acc[i] = __builtin_fmaf(wj[j], (float)v[j].v[i], acc[i]);
    }
    g53_store8_to(out + t * H, acc, c, H);
}

static int combine(const char *who, void *out, const void *ys, const float *w, const void *add, int dt, int hidden,
                   const G53hSort *p)
{
    if (g53h_ready()) return -1;
    const int chunks = (hidden + 2047) / 2048;
    const long total = (long)p->T * chunks;
    for (long w0 = 0; w0 < total; w0 += G53_LAUNCH_WGS) {
        const unsigned wgs = (unsigned)(total - w0 < G53_LAUNCH_WGS ? total - w0 : G53_LAUNCH_WGS);
        G53_BY_TYPE(dt, hipLaunchKernelGGL(k_sorted_combine<E>, dim3(wgs), dim3(256), 0, g53h_stream(), (E *)out, (const E *)ys, w,
                                           (const E *)add, p->row, hidden, p->topk, chunks, w0));
        G53_LAUNCHED("k_sorted_combine");
    }
    return 0;
}

extern "C" int g53h_sorted_combine(void *out, const void *ys, const float *w, const void *add, int dt, int hidden,
                                   const G53hSort *p)
{
    if (rows_bad("g53h_sorted_combine", p, dt, hidden)) return -1;
    if (!p->T) return 0;
    if (!out || !ys || !w) return g53h_fail("g53h_sorted_combine: no rows or no weights");
    return combine("g53h_sorted_combine", out, ys, w, add, dt, hidden, p);
}

extern "C" int g53h_sorted_dispatch_grad(void *dx, const void *dxs, int dt, int hidden, const G53hSort *p)
{
    if (rows_bad("g53h_sorted_dispatch_grad", p, dt, hidden)) return -1;
    if (!p->T) return 0;
    if (!dx || !dxs) return g53h_fail("g53h_sorted_dispatch_grad: no rows");
    return combine("g53h_sorted_dispatch_grad", dx, dxs, nullptr, nullptr, dt, hidden, p);
}

/* One wave per pair: dys of its row, dw of the pair. */
template <typename E>
__global__ void __launch_bounds__(256)
k_sorted_combine_grad(E *dys, float *__restrict__ dw, const E *__restrict__ dout, const E *ys, const float *__restrict__ w,
               const int *__restrict__ row, int H, int K, long n, long wg0)
{
    const int lane = threadIdx.x & 63;
    const long p = (wg0 + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (p >= n) return;
    const long r = row[p];
    if (r < 0) {
        if (lane == 0) dw[p] = 0.0f;
        return;
    }
    const float wp = w[p];
    const E *g = dout + p / K * H, *y = ys + r * H;
    E *d = dys + r * H;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int c = lane * 8; c < H; c += 512) {
        float gv[8], o[8];
        G53Raw8<E> yv;
        g53_load8_to(gv, g, c, H);
        g53_raw8_once_to(yv, y, c, H);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            acc[i] = __builtin_fmaf(gv[i], (float)yv.v[i], acc[i]);
            o[i] = wp * gv[i];
        }
        g53_store8_to(d, o, c, H);
    }
    const float s = g53_wave_sum(((acc[0] + acc[4]) + (acc[2] + acc[6])) + ((acc[1] + acc[5]) + (acc[3] + acc[7])));
    if (lane == 0) dw[p] = s;
}

extern "C" int g53h_sorted_combine_grad(void *dys, float *dw, const void *dout, const void *ys, const float *w, int dt,
                                        int hidden, const G53hSort *p)
{
    if (rows_bad("g53h_sorted_combine_grad", p, dt, hidden)) return -1;
    if (!p->T) return 0;
    if (!dys || !dw || !dout || !ys || !w) return g53h_fail("g53h_sorted_combine_grad: no rows or no weights");
    if (g53h_ready()) return -1;
    const long n = (long)p->T * p->topk, total = (n + 3) / 4;
    for (long w0 = 0; w0 < total; w0 += G53_LAUNCH_WGS) {
        const unsigned wgs = (unsigned)(total - w0 < G53_LAUNCH_WGS ? total - w0 : G53_LAUNCH_WGS);
        G53_BY_TYPE(dt, hipLaunchKernelGGL(k_sorted_combine_grad<E>, dim3(wgs), dim3(256), 0, g53h_stream(), (E *)dys, dw,
                                           (const E *)dout, (const E *)ys, w, p->row, hidden, p->topk, n, w0));
        G53_LAUNCHED("k_sorted_combine_grad");
    }
    return 0;
}
