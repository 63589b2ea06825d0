/* g53h_norm.hip - the norms before and after a block, fused with the block's gate and residual
 * scale, and their gradients.
 *
 *     u  = y / sqrt(mean y^2 + eps) * post        (post NULL: u = y)
 *     h' = h + scale * gate * u
 *     xn = h' / sqrt(mean h'^2 + eps) * next
 *
 * and, with rs = 1 / sqrt(mean^2 + eps) and a hat for a value times its rs,
 *
 *     v  = dxn next,   dH = dh' + rs(h') (v - h'^ mean(v h'^)),   dnext = sum over tokens of dxn h'^
 *     dh = dH,   dgate = scale u dH summed over what shares the gate
 *     du = scale gate dH,   dpost = sum over tokens of du y^
 *     dy = rs(y) (du post - y^ mean(du post y^))
 *
 * Both directions are one pass over HBM: W waves hold a token's row in registers, 8 elements a lane
 * (16 for rows above 4096, 32 above 8192), sums go over the lanes and then the waves. The next norm takes h' in fp32,
 * before it is rounded to be stored, and the backward pass forms that h' again from h and y, with roundings of its own
 * (a last bit of fp32 may differ).
 * Gradients that tokens share are summed by each workgroup over its tokens in registers, written once
 * and added up by k_norm_sum in a fixed order: no atomics, the same bits on every run.
 *
 * Both are bound by HBM once there are many tokens: forward 8192 x 4096 bf16 with a gate per channel 55.5 us,
 * 4.8 TB/s, backward 4096 x 4096 44 us, 4.6 TB/s with the sums' launch (4 us). A gradient of few tokens is
 * latency: two launches, a workgroup a CU that meets memory, two sums over its waves and one barrier each per
 * token, and as many bytes of partial sums as of two rows a workgroup (1025 x 4096: 14 us and 4, floor 10.6).
 * Gradients with a block output spill above 4096 wide: 10 to 42 registers up to 8192 (1024 x 8192 bf16: 40 us,
 * floor 21), 158 to 324 above (512 x 16384: 92, floor 21); without one, 4 in fp32 above 8192 (22, floor 10.6, in bf16).
 */
#include <hip/hip_runtime.h>

#include "g53h.h"
#include "g53h_elem.h"
#include "g53h_runtime.h"

#define G53_NORM_MAXH 16384

struct G53NormArgs {
    const float *post, *next;
    const void *gate;                   /* kind 1: float [H], 2: float [T], 3: E [T][H] */
    void *dgate;                        /* kinds 2 and 3 */
    float *part;                        /* partial sums [workgroups][2][pitch] of dpost over scale and channel's gate, and dnext */
    float eps, scale;
    int T, H, pitch;                    /* H up to a multiple of 32 */
};

/* 1 / sqrt(v), off by one in the last place at most; v is at least eps, a normal number. */
__device__ __forceinline__ float g53_rsq(float v) { return __builtin_amdgcn_rsqf(v); }

/* Sums of N values over the W waves of a row's group, in every lane; buf: N floats a wave. */
template <int W, int N> __device__ __forceinline__ void g53_group_sum(float (&v)[N], float (*buf)[N], int wv)
{
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = g53_wave_sum(v[k]);
    if (W > 1) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; k++) buf[wv][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; k++) {
            v[k] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) v[k] += buf[wv / W * W + w][k];
        }
    }
}

/* GK: the gate's kind; Y: there is a block output (else the norm of h alone). */
template <typename E, int W, int NV, int GK, bool Y>
__global__ void __launch_bounds__(W < 4 ? 256 : 64 * W)
k_block_norm(E *h2, E *xn, const E *h, const E *y, G53NormArgs a, long wg0)
{
    constexpr int NW = W < 4 ? 4 : W, RB = NW / W;
    __shared__ float buf[2][NW][1];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    long t = (wg0 + blockIdx.x) * RB + wv / W;
    const bool live = t < a.T;
    if (!live) t = a.T - 1;             /* rows behind the last: computed, not written */
    const int H = a.H, c0 = ((wv % W) * 64 + lane) * 8;
    float hv[NV][8], s[1] = {0.0f};
    float pv[NV][8], gv[NV][8], nv[NV][8];
    constexpr bool EARLY = NV == 1;     /* gains are asked for with the rows */
    auto gains = [&](int v) {
        const int c = c0 + v * 512 * W;
        if (Y && a.post) g53_load8_to(pv[v], a.post, c, H);
        if (Y && GK == 1) g53_load8_to(gv[v], (const float *)a.gate, c, H);
        if (Y && GK == 3) g53_load8_to(gv[v], (const E *)a.gate + t * H, c, H);
    };
    auto next = [&](int v) {
        if (xn) g53_load8_to(nv[v], a.next, c0 + v * 512 * W, H);
    };
#pragma unroll
    for (int v = 0; v < NV; v++) g53_load8_to(hv[v], h + t * H, c0 + v * 512 * W, H);
    if (Y) {
        float yv[NV][8];
#pragma unroll
        for (int v = 0; v < NV; v++) g53_load8_to(yv[v], y + t * H, c0 + v * 512 * W, H);
        if (EARLY) {
            gains(0);
            next(0);
        }
        float rs = 1.0f;
        if (a.post) {
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) s[0] = __builtin_fmaf(yv[v][i], yv[v][i], s[0]);
            g53_group_sum<W, 1>(s, buf[0], wv);
            rs = g53_rsq(s[0] / (float)H + a.eps);
        }
        const float gt = a.scale * (GK == 2 ? ((const float *)a.gate)[t] : 1.0f);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = c0 + v * 512 * W;
            if (!EARLY) gains(v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float u = a.post ? yv[v][i] * rs * pv[v][i] : yv[v][i];
                hv[v][i] = __builtin_fmaf((GK & 1) ? gt * gv[v][i] : gt, u, hv[v][i]);
            }
            if (live) g53_store8_to(h2 + t * H, hv[v], c, H);
        }
    } else if (EARLY) {
        next(0);
    }
    if (!xn) return;
    s[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
        for (int i = 0; i < 8; i++) s[0] = __builtin_fmaf(hv[v][i], hv[v][i], s[0]);
    g53_group_sum<W, 1>(s, buf[1], wv);
    const float rs = g53_rsq(s[0] / (float)H + a.eps);
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int c = c0 + v * 512 * W;
        if (!EARLY) next(v);
#pragma unroll
        for (int i = 0; i < 8; i++) hv[v][i] = hv[v][i] * rs * nv[v][i];
        if (live) g53_store8_to(xn + t * H, hv[v], c, H);
    }
}

/* Persistent: group g of W waves takes tokens g, g + groups, ...; the next token's rows are asked for before a token's sums
 * where registers hold them (rows of up to 4096).
 * With k = scale gate post two rounds of sums are enough: y's squares, then h''s squares and its products with v and k y^,
 * and k y^'s with v and dh', from which mean(v h'^) and mean(du post y^) = mean(k y^ dH) follow. Where the gate is the same for
 * all tokens (kinds 0 and 1), A = sum over tokens of y^ dH gives dpost = scale gate A and dgate = scale post A. */
template <typename E, int W, int NV, int GK, bool Y>
__global__ void __launch_bounds__(W < 4 ? 256 : 64 * W)
k_block_norm_grad(E *dh, E *dy, const E *dh2, const E *dxn, const E *h, const E *y, G53NormArgs a)
{
    constexpr int NW = W < 4 ? 4 : W, RB = NW / W;
    constexpr bool KEEP = NV == 1;             /* gains stay in registers, and the next token's rows wait there */
    constexpr bool HELD = NV < 4;               /* sums over tokens too; of rows above 8192 they are in LDS */
    __shared__ float buf1[2][NW][1], buf2[2][NW][5];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long grp = (long)blockIdx.x * RB + wv / W, groups = (long)gridDim.x * RB;
    const int H = a.H, c0 = ((wv % W) * 64 + lane) * 8;
    const long rounds = (a.T + groups - 1) / groups;
    const float inv = 1.0f / (float)H;
    float ap[NV][8], an[NV][8];
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float *sums = (float *)lds + threadIdx.x * 4;    /* [2][NV][2][threads][4], HELD false */
    auto at = [&](int which, int v, int b) { return (g53_v4f *)(sums + ((which * NV + v) * 2 + b) * (64 * NW * 4)); };
    auto add = [&](float (&to)[NV][8], int which, int v, const float (&p)[8], const float (&q)[8]) {   /* of p q */
        if (HELD) {
#pragma unroll
            for (int i = 0; i < 8; i++) to[v][i] = __builtin_fmaf(p[i], q[i], to[v][i]);
        } else {
#pragma unroll
            for (int b = 0; b < 2; b++) {
                g53_v4f o = *at(which, v, b);
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(p[4 * b + i], q[4 * b + i], o[i]);
                *at(which, v, b) = o;
            }
        }
    };
    float kp[NV][8], kn[NV][8];                /* scale gate post, or scale post for kinds 2 and 3; next */
    auto gains = [&](int v) {
        const int c = c0 + v * 512 * W;
        float gv[8];                                 /* all asked for before the first is used */
#pragma unroll
        for (int i = 0; i < 8; i++) { kp[v][i] = 1.0f; kn[v][i] = 0.0f; }
        if (dxn) g53_load8_to(kn[v], a.next, c, H);
        if (Y && a.post) g53_load8_to(kp[v], a.post, c, H);
        if (Y && GK == 1) g53_load8_to(gv, (const float *)a.gate, c, H);
#pragma unroll
        for (int i = 0; i < 8; i++) kp[v][i] *= Y && GK == 1 ? a.scale * gv[i] : a.scale;
    };
    G53Raw8<E> rh[NV], ry[NV], rg[NV], rd[NV], rt[NV];
    float rgate = 1.0f;
    auto ask = [&](long t) {                         /* behind the last token: the group's own last again, not used */
        if (t >= a.T) t = t >= groups && t - groups < a.T ? t - groups : a.T - 1;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = c0 + v * 512 * W;
            if (Y) g53_raw8_to(ry[v], y + t * H, c, H);
            g53_raw8_to(rh[v], h + t * H, c, H);
            if (dxn) g53_raw8_to(rd[v], dxn + t * H, c, H);
            if (dh2) g53_raw8_to(rg[v], dh2 + t * H, c, H);
            if (Y && GK == 3) g53_raw8_to(rt[v], (const E *)a.gate + t * H, c, H);
        }
        if (Y && GK == 2) rgate = ((const float *)a.gate)[t];
    };
    if (KEEP) ask(grp);
#pragma unroll
    for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int i = 0; i < 8; i++) ap[v][i] = an[v][i] = 0.0f;
        if (!HELD)
#pragma unroll
            for (int k = 0; k < 4; k++) *at(k >> 1, v, k & 1) = (g53_v4f){0.0f, 0.0f, 0.0f, 0.0f};
        if (KEEP) gains(v);
    }
    for (long r = 0; r < rounds; r++) {
        const long t = grp + r * groups;
        const bool live = t < a.T;
        if (!KEEP) ask(t);
        const int odd = r & 1;                       /* sums of two tokens in a row lie apart: one barrier each is enough */
        float hv[NV][8], yh[NV][8], g_[NV][8], d_[NV][8], w[NV][8], gt_[NV][8];
        const float tgate = rgate;
        /* dh', dxn and the gate of the element: in fp32 where the next token's take their place, else as they came */
        auto g = [&](int v, int i) { return KEEP ? g_[v][i] : dh2 ? (float)rg[v].v[i] : 0.0f; };
        auto d = [&](int v, int i) { return KEEP ? d_[v][i] : dxn ? (float)rd[v].v[i] : 0.0f; };
        auto gt = [&](int v, int i) { return KEEP ? gt_[v][i] : (float)rt[v].v[i]; };
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                hv[v][i] = (float)rh[v].v[i];
                if (Y) yh[v][i] = (float)ry[v].v[i];
                if (KEEP) d_[v][i] = dxn ? (float)rd[v].v[i] : 0.0f;
                if (KEEP) g_[v][i] = dh2 ? (float)rg[v].v[i] : 0.0f;
                if (KEEP && Y && GK == 3) gt_[v][i] = (float)rt[v].v[i];
            }
        if (KEEP) ask(t + groups);
        float rsy = 1.0f;
        if (Y && a.post) {
            float s[1] = {0.0f};
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) s[0] = __builtin_fmaf(yh[v][i], yh[v][i], s[0]);
            g53_group_sum<W, 1>(s, buf1[odd], wv);
            rsy = g53_rsq(s[0] * inv + a.eps);
        }
        /* the factor of y^ in h', of dH in dy */
        auto factor = [&](int v, int i) { return GK < 2 ? kp[v][i] : kp[v][i] * (GK == 2 ? tgate : gt(v, i)); };
        float s[5] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < NV; v++) {
            if (!KEEP) gains(v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[v][i] = d(v, i) * kn[v][i];
                if (Y) {
                    yh[v][i] *= rsy;
                    const float u = factor(v, i) * yh[v][i];
                    hv[v][i] += u;
                    s[2] = __builtin_fmaf(u, g(v, i), s[2]);
                    s[3] = __builtin_fmaf(u, w[v][i], s[3]);
                    s[4] = __builtin_fmaf(u, hv[v][i], s[4]);
                }
                s[0] = __builtin_fmaf(hv[v][i], hv[v][i], s[0]);
                s[1] = __builtin_fmaf(w[v][i], hv[v][i], s[1]);
            }
        }
        g53_group_sum<W, 5>(s, buf2[odd], wv);
        const float rs = dxn ? g53_rsq(s[0] * inv + a.eps) : 0.0f, mean = s[1] * rs * inv;
        const float to_y = a.post ? -rsy * (s[2] + rs * (s[3] - rs * mean * s[4])) * inv : 0.0f;
        float gsum[1] = {0.0f};
        if (KEEP)                                   /* the next token's rows, before this one's stores */
#pragma unroll
            for (int v = 0; v < NV; v++) {
                g53_arrived(rh[v]);
                if (Y) g53_arrived(ry[v]);
                if (dxn) g53_arrived(rd[v]);
                if (dh2) g53_arrived(rg[v]);
                if (Y && GK == 3) g53_arrived(rt[v]);
            }
        if (live)
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = c0 + v * 512 * W;
                float dg[8], dv[8], o[8];
                if (!KEEP) {                         /* converted again, not kept in fp32 */
                    if (dxn) g53_arrived(rd[v]);
                    if (dh2) g53_arrived(rg[v]);
                    if (Y && GK == 3) g53_arrived(rt[v]);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    hv[v][i] *= rs;
                    dv[i] = d(v, i);
                    o[i] = __builtin_fmaf(rs, __builtin_fmaf(-hv[v][i], mean, w[v][i]), g(v, i));
                }
                add(an, 1, v, dv, hv[v]);
                g53_store8_to(dh + t * H, o, c, H);
                if (!Y) continue;
                if (GK < 2) add(ap, 0, v, yh[v], o);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (GK >= 2) {
                        const float yg = yh[v][i] * o[i];
                        dv[i] = GK == 2 ? tgate : gt(v, i);
                        dg[i] = kp[v][i] * yg;
                        gsum[0] += dg[i];
                        hv[v][i] = yg;
                    }
                    o[i] = __builtin_fmaf(to_y, yh[v][i], rsy * (factor(v, i) * o[i]));      /* without post: du itself */
                }
                if (GK >= 2) add(ap, 0, v, dv, hv[v]);
                if (GK == 3 && a.dgate) g53_store8_to((E *)a.dgate + t * H, dg, c, H);
                g53_store8_to(dy + t * H, o, c, H);
            }
        if (Y && GK == 2 && a.dgate) {
            __shared__ float bufg[2][NW][1];
            g53_group_sum<W, 1>(gsum, bufg[odd], wv);
            if (live && lane == 0 && wv % W == 0) ((float *)a.dgate)[t] = gsum[0];
        }
    }
    /* the sums of the workgroup's groups, added in order by the first of them, which writes them */
    float *part = a.part + (long)blockIdx.x * 2 * a.pitch;
    auto finish = [&](float (&v8)[NV][8], int which) {
        if (!HELD)
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) v8[v][i] = (*at(which, v, i >> 2))[i & 3];
        if (RB > 1) {                                /* NV = 1 */
            __shared__ float rows[RB > 1 ? NW : 1][8][64];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; i++) rows[wv][i][lane] = v8[0][i];
            __syncthreads();
            if (wv >= W) return;
#pragma unroll
            for (int r = 1; r < RB; r++)
#pragma unroll
                for (int i = 0; i < 8; i++) v8[0][i] += rows[r * W + wv][i][lane];
        }
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = c0 + v * 512 * W;
            if (c < a.pitch) g53_store8(part + which * a.pitch + c, v8[v]);    /* zeros behind H */
        }
    };
    if (Y) finish(ap, 0);
    finish(an, 1);
}

/* 32 columns of the workgroups' partial sums, added in a fixed order: 32 chains, four columns a lane, then a tree. The
 * first sums give dpost and the gradient of a gate by channel (scale and the other's value times the sum; the gate by
 * token or element is in it already), the second dnext. */
__global__ void __launch_bounds__(256) k_norm_sum(float *__restrict__ dpost, float *__restrict__ dnext, float *__restrict__ dgate,
                                                  const float *__restrict__ post, const float *__restrict__ gate,
                                                  const float *__restrict__ part, float scale, int parts, int H, int pitch)
{
    __shared__ g53_v4f buf[4][8];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, which = blockIdx.y;
    if (which ? !dnext : !dpost && !dgate) return;
    const float *from = part + which * pitch + blockIdx.x * 32 + (lane & 7) * 4;
    g53_v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int g = wv * 8 + (lane >> 3); g < parts; g += 32) {
        const g53_v4f v = *(const g53_v4f *)(from + (long)g * 2 * pitch);
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] += v[i];
    }
#pragma unroll
    for (int d = 8; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] += __shfl_xor(s[i], d);
    if (lane < 8) buf[wv][lane] = s;
    __syncthreads();
    const int c = blockIdx.x * 32 + threadIdx.x;
    if (threadIdx.x >= 32 || c >= H) return;
    const float *b = (const float *)buf + threadIdx.x;
    const float t = (b[0] + b[32]) + (b[64] + b[96]);
    if (which) {
        dnext[c] = t;
        return;
    }
    if (dpost) dpost[c] = scale * (gate ? gate[c] : 1.0f) * t;
    if (dgate) dgate[c] = scale * (post ? post[c] : 1.0f) * t;
}

/* Waves per row: 512 elements each up to 4096, then eight with more. Of 16 the gradient's registers do not hold the rows
 * (1024 x 8192 bf16: 82 us against 38; 512 x 16384, sums in registers: 155 against 93). */
#define G53_NORM_BY_WIDTH(H, BODY)                                              \
    do {                                                                        \
        if ((H) <= 512) { constexpr int W = 1, NV = 1; BODY; }                  \
        else if ((H) <= 1024) { constexpr int W = 2, NV = 1; BODY; }            \
        else if ((H) <= 2048) { constexpr int W = 4, NV = 1; BODY; }            \
        else if ((H) <= 4096) { constexpr int W = 8, NV = 1; BODY; }            \
        else if ((H) <= 8192) { constexpr int W = 8, NV = 2; BODY; }            \
        else { constexpr int W = 8, NV = 4; BODY; }                             \
    } while (0)
#define G53_NORM_BY_GATE(kind, BODY)                                            \
    do {                                                                        \
        if ((kind) == 0) { constexpr int GK = 0; BODY; }                        \
        else if ((kind) == 1) { constexpr int GK = 1; BODY; }                   \
        else if ((kind) == 2) { constexpr int GK = 2; BODY; }                   \
        else { constexpr int GK = 3; BODY; }                                    \
    } while (0)

#define G53_NORM_WGS (1l << 21)         /* workgroups of one launch: of up to 1024 threads, counted in 32 bits */

template <typename E, int W, int NV, int GK, bool Y>
static int forward(void *h2, void *xn, const void *h, const void *y, const G53NormArgs &a)
{
    constexpr int NW = W < 4 ? 4 : W, RB = NW / W;
    const long total = ((long)a.T + RB - 1) / RB;
    for (long w0 = 0; w0 < total; w0 += G53_NORM_WGS) {
        const unsigned wgs = (unsigned)(total - w0 < G53_NORM_WGS ? total - w0 : G53_NORM_WGS);
        hipLaunchKernelGGL((k_block_norm<E, W, NV, GK, Y>), dim3(wgs), dim3(64 * NW), 0, g53h_stream(), (E *)h2, (E *)xn,
                           (const E *)h, (const E *)y, a, w0);
        G53_LAUNCHED("k_block_norm");
    }
    return 0;
}

template <typename E, int W, int NV, int GK, bool Y>
static int backward(void *dh, void *dy, float *dpost, float *dnext, float *dchannel, const void *dh2, const void *dxn,
                    const void *h, const void *y, G53NormArgs &a)
{
    constexpr int NW = W < 4 ? 4 : W, RB = NW / W;
    /* eight waves a CU, all with the same number of tokens where that divides */
    const long most = g53h_num_cus() * (W < 8 ? 2 : 1), need = ((long)a.T + RB - 1) / RB, rounds = (need + most - 1) / most;
    const unsigned wgs = (unsigned)(need ? (need + rounds - 1) / rounds : 0);
    constexpr size_t lds = NV < 4 ? 0 : (size_t)4 * NV * 64 * NW * sizeof(g53_v4f);
    if (wgs) {
        static int allowed = 0;
        if (lds && !allowed) {
            G53_TRY(hipFuncSetAttribute((const void *)k_block_norm_grad<E, W, NV, GK, Y>,
                                        hipFuncAttributeMaxDynamicSharedMemorySize, lds));
            allowed = 1;
        }
        a.part = (float *)g53h_op_workspace((size_t)wgs * 2 * a.pitch * sizeof(float));
        if (!a.part) return -1;
        hipLaunchKernelGGL((k_block_norm_grad<E, W, NV, GK, Y>), dim3(wgs), dim3(64 * NW), lds, g53h_stream(), (E *)dh, (E *)dy,
                           (const E *)dh2, (const E *)dxn, (const E *)h, (const E *)y, a);
        G53_LAUNCHED("k_block_norm_grad");
    }
    if (dpost || dnext || dchannel) {
        hipLaunchKernelGGL(k_norm_sum, dim3(a.pitch / 32, 2), dim3(256), 0, g53h_stream(), dpost, dnext, dchannel, a.post,
                           GK == 1 ? (const float *)a.gate : nullptr, a.part, a.scale, (int)wgs, a.H, a.pitch);
        G53_LAUNCHED("k_norm_sum");
    }
    return 0;
}

static int norm_bad(const char *who, int T, int hidden, int dt, float eps)
{
    if (T < 0 || hidden < 1 || hidden > G53_NORM_MAXH || !g53_elem_bytes(dt))
        return g53h_fail("%s: %d tokens of %d, element type %d (hidden at most %d)", who, T, hidden, dt, G53_NORM_MAXH);
    if (!(eps >= 1.0e-30f) || eps > 1.0e30f) return g53h_fail("%s: eps %g (1e-30 to 1e30)", who, eps);
    return 0;
}

static int block_bad(const char *who, const G53hBlockNorm *p, G53NormArgs &a)
{
    if (!p) return g53h_fail("%s: no parameters", who);
    if (norm_bad(who, p->T, p->hidden, p->dt, p->eps)) return -1;
    if (p->gate_kind < 0 || p->gate_kind > 3 || (p->gate_kind && p->T && !p->gate))
        return g53h_fail("%s: gate kind %d%s", who, p->gate_kind, p->gate ? "" : ", no gate");
    if (!(p->scale >= -1.0e30f && p->scale <= 1.0e30f)) return g53h_fail("%s: scale %g", who, p->scale);
    a = G53NormArgs{p->post, p->next, p->gate, nullptr, nullptr, p->eps, p->scale, p->T, p->hidden, (p->hidden + 31) & ~31};
    return 0;
}

extern "C" int g53h_norm(void *xn, const void *x, const float *gain, int dt, int T, int hidden, float eps)
{
    if (norm_bad("g53h_norm", T, hidden, dt, eps)) return -1;
    if (!T) return 0;
    if (!xn || !x || !gain) return g53h_fail("g53h_norm: no rows or no gain");
    if (g53h_ready()) return -1;
    G53NormArgs a{nullptr, gain, nullptr, nullptr, nullptr, eps, 0.0f, T, hidden, (hidden + 31) & ~31};
    int rc;
    G53_BY_TYPE(dt, G53_NORM_BY_WIDTH(hidden, rc = (forward<E, W, NV, 0, false>(nullptr, xn, x, nullptr, a))));
    return rc;
}

extern "C" int g53h_norm_grad(void *dx, float *dgain, const void *dxn, const void *x, const float *gain, int dt, int T,
                              int hidden, float eps)
{
    if (norm_bad("g53h_norm_grad", T, hidden, dt, eps)) return -1;
    if (T && (!dx || !dxn || !x || !gain)) return g53h_fail("g53h_norm_grad: no rows or no gain");
    if (g53h_ready()) return -1;
    G53NormArgs a{nullptr, gain, nullptr, nullptr, nullptr, eps, 0.0f, T, hidden, (hidden + 31) & ~31};
    int rc;
    G53_BY_TYPE(dt, G53_NORM_BY_WIDTH(hidden, rc = (backward<E, W, NV, 0, false>(dx, nullptr, nullptr, dgain, nullptr, nullptr,
                                                                                  dxn, x, nullptr, a))));
    return rc;
}

extern "C" int g53h_block_norm(void *h2, void *xn, const void *h, const void *y, const G53hBlockNorm *p)
{
    G53NormArgs a;
    if (block_bad("g53h_block_norm", p, a)) return -1;
    if (!p->T) return 0;
    if (!h2 || !h || !y) return g53h_fail("g53h_block_norm: no rows");
    if (xn && !p->next) return g53h_fail("g53h_block_norm: xn without its gain");
    if (g53h_ready()) return -1;
    int rc;
    G53_BY_TYPE(p->dt, G53_NORM_BY_WIDTH(p->hidden, G53_NORM_BY_GATE(p->gate_kind,
                rc = (forward<E, W, NV, GK, true>(h2, xn, h, y, a)))));
    return rc;
}

extern "C" int g53h_block_norm_grad(void *dh, void *dy, void *dgate, float *dpost, float *dnext, const void *dh2,
                                    const void *dxn, const void *h, const void *y, const G53hBlockNorm *p)
{
    G53NormArgs a;
    if (block_bad("g53h_block_norm_grad", p, a)) return -1;
    if (p->T && (!dh || !dy || !h || !y)) return g53h_fail("g53h_block_norm_grad: no rows");
    if (p->T && !dh2 && !dxn) return g53h_fail("g53h_block_norm_grad: neither dh2 nor dxn");
    if (dxn && !p->next) return g53h_fail("g53h_block_norm_grad: dxn without its gain");
    if (g53h_ready()) return -1;
    if (!p->post) dpost = nullptr;
    if (!p->next) dnext = nullptr;
    a.dgate = p->gate_kind >= 2 ? dgate : nullptr;
    float *dchannel = p->gate_kind == 1 ? (float *)dgate : nullptr;
    int rc;
    G53_BY_TYPE(p->dt, G53_NORM_BY_WIDTH(p->hidden, G53_NORM_BY_GATE(p->gate_kind,
                rc = (backward<E, W, NV, GK, true>(dh, dy, dpost, dnext, dchannel, dh2, dxn, h, y, a)))));
    return rc;
}
