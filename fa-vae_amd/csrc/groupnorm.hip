// Group norm with an activation over channels-last maps, forward and backward.
//
//   per sample n and group g, over the m = S * Cg values of its S positions and Cg channels:
//     mean = sum x / m,  rstd = (sum (x - mean)^2 / m + eps)^-1/2,  xh = (x - mean) rstd,  z = gamma xh + beta,  y = act(z)
//   backward:  dz = dy act'(z),  dbeta = sum dz,  dgamma = sum dz xh  (over samples and positions),
//     dx = rstd (gamma dz - (s1 + xh s2) / m),  s1 = sum over the group of gamma dz,  s2 = sum over the group of gamma dz xh
//   The kernels work with d = x - mean: z = fma(d, gamma rstd, beta), sum dz d, and dx = (gamma rstd) dz - c1 - d c2 with
//   c1 = rstd s1 / m, c2 = rstd^2 s2 / m.
//
// Memory bounds both.  Held form: one workgroup holds all positions of a run of whole groups in registers, so that the input is read
// once: load, sum, sum of squared distances from the mean (no cancellation), normalise, store.  Chunked form, where a group is too
// large for one workgroup's registers or there are too few groups to fill the chip: a first launch leaves the partial sums of each
// chunk of positions, a second one joins them and makes the pass over the data.  Sums are fp32 within a chunk and joined in a fixed
// order: the results do not depend on scheduling.
#include "groupnorm.h"
#include <numeric>

namespace {

// ---- forward -------------------------------------------------------------------------------------------------------------
// STATS: leave (mean, sum of squared distances) of this chunk in part[((n G + g) nchunk + chunk) pieces + piece] and stop.
template <class T, int VEC, int ITEMS, bool GS, bool STATS> __global__ __launch_bounds__(GTF) void gn_fwd_kernel(const GnP p) {
    extern __shared__ float lds[];
    constexpr int NV = GS ? 1 : VEC;
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const int chunk = (int)(t_ % p.nchunk);
    const long long nb0 = t_ / p.nchunk;
    const GnBlock b = gn_block(p, cb);
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int sub = r / p.P, pos = r - sub * p.P;
    const long long n = nb0 * p.NSUB + sub;
    const int c0 = b.c_lo + lv * VEC;
    const int s_lo = chunk * p.chunk, s_hi = min(p.S, s_lo + p.chunk);
    const bool active = sub < p.NSUB && n < p.N && c0 < b.c_hi;
    float* red = lds;
    float* grp = lds + GTF * NV;

    GnData<T, VEC> d[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int s = s_lo + pos + i * p.P;
        if (active && s < s_hi) d[i].load(p.x, n * p.xn + s * p.xs + c0);
    }
    float v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (active && s_lo + pos + i * p.P < s_hi) {
            float f[VEC];
            d[i].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[GS ? 0 : j] += f[j];
            d[i].keep();
        }
    }
    const int cpg = GS ? b.cw / VEC : b.cw;
    gn_reduce<NV>(p, v, red, grp, lv, r, b.ng, cpg);
    const float inv = s_hi > s_lo ? 1.f / ((float)(s_hi - s_lo) * (float)b.cw) : 0.f;
    GnStat<VEC, GS> st;
    int gl[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        gl[j] = active ? sub * b.ng + (p.pieces == 1 ? (lv * VEC + j) / p.Cg : 0) : 0;
        st.m[j] = grp[gl[j]] * inv;
        v[j] = 0.f;
    }
    float keep_mean = 0.f;                       // a pair's mean, by the thread that stores it
    const int pairs = p.NSUB * b.ng;
    if ((int)threadIdx.x < pairs && pairs <= GTF) keep_mean = grp[threadIdx.x] * inv;
    if (pairs > GTF)                              // more pairs than threads: through memory at once (grp is reused below)
        for (int k = threadIdx.x; k < pairs; k += GTF) {
            const long long nn = nb0 * p.NSUB + k / b.ng;
            if (nn < p.N) {
                if constexpr (STATS) p.part[((nn * p.G + b.g_lo + k % b.ng) * p.nchunk + chunk) * p.pieces + b.piece].x = grp[k] * inv;
                else p.mean[nn * p.G + b.g_lo + k % b.ng] = grp[k] * inv;
            }
        }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (active && s_lo + pos + i * p.P < s_hi) {
            float f[VEC];
            d[i].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) { const float t = f[j] - st.mean(j); v[GS ? 0 : j] = fmaf(t, t, v[GS ? 0 : j]); }
            d[i].keep();
        }
    }
    gn_reduce<NV>(p, v, red, grp, lv, r, b.ng, cpg);
    for (int k = threadIdx.x; k < pairs; k += GTF) {
        const long long nn = nb0 * p.NSUB + k / b.ng;
        const int g = b.g_lo + k % b.ng;
        if (nn < p.N) {
            if constexpr (STATS) {
                float2* o = p.part + ((nn * p.G + g) * p.nchunk + chunk) * p.pieces + b.piece;
                if (pairs <= GTF) o->x = keep_mean;
                o->y = grp[k];
            } else {
                if (pairs <= GTF) p.mean[nn * p.G + g] = keep_mean;
                p.rstd[nn * p.G + g] = 1.f / sqrtf(grp[k] * inv + p.eps);
            }
        }
    }
    if constexpr (!STATS) {
        if (!active) return;
        float ga[VEC], be[VEC];
#pragma unroll
        for (int j = 0; j < NV; ++j) st.r[j] = 1.f / sqrtf(grp[gl[j]] * inv + p.eps);
#pragma unroll
        for (int j = 0; j < VEC; ++j) { ga[j] = p.gamma[c0 + j] * st.rstd(j); be[j] = p.beta[c0 + j]; }
        if constexpr (VEC * sizeof(T) == 16) {
            if (p.qo) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const int s = s_lo + pos + i * p.P;
                    if (s < s_hi) {
                        float f[VEC];
                        d[i].get(f);
                        ck_store<VEC>(p, f, n * p.S + s, c0);
                    }
                }
            }
        }
        with_act(p.act, [&](auto a) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int s = s_lo + pos + i * p.P;
                if (s < s_hi) {
                    float f[VEC];
                    d[i].get(f);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] = fmaf(f[j] - st.mean(j), ga[j], be[j]);
                    act_apply<T, decltype(a)::value>(f);
                    typename VecOf<T, VEC>::raw o;
                    vec_put(o, f);
                    *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
                }
            }
        });
    }
}

// Chunked form, second launch: join the chunks of this block's groups (mean of means, and sums of squared distances moved to it), normalise.
template <class T, int VEC, bool GS> __global__ __launch_bounds__(GTF) void gn_apply_kernel(const GnP p) {
    extern __shared__ float lds[];
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const int chunk = (int)(t_ % p.nchunk);
    const long long n = t_ / p.nchunk;
    const GnBlock b = gn_block(p, cb);
    const int parts = p.nchunk * p.pieces;
    float2* stat = (float2*)lds;                 // [ng] (mean, rstd)
    for (int g = threadIdx.x >> 6; g < b.ng; g += GTF / 64) {
        const float2* a = p.part + (n * p.G + b.g_lo + g) * parts;
        const float m = (float)p.S * (float)p.Cg;
        float s = 0.f, q = 0.f;
        for (int i = threadIdx.x & 63; i < parts; i += 64) {
            const int ch = i / p.pieces, pc = i - ch * p.pieces;
            const float cnt = (float)(min(p.S, (ch + 1) * p.chunk) - ch * p.chunk) * (float)(p.pieces == 1 ? p.Cg : min(p.Cg, (pc + 1) * p.CB) - pc * p.CB);
            s = fmaf(cnt, a[i].x, s);
        }
        const float mean = wave_total(s) / m;
        for (int i = threadIdx.x & 63; i < parts; i += 64) {
            const int ch = i / p.pieces, pc = i - ch * p.pieces;
            const float cnt = (float)(min(p.S, (ch + 1) * p.chunk) - ch * p.chunk) * (float)(p.pieces == 1 ? p.Cg : min(p.Cg, (pc + 1) * p.CB) - pc * p.CB);
            const float dm = a[i].x - mean;
            q += fmaf(cnt * dm, dm, a[i].y);
        }
        const float rstd = 1.f / sqrtf(wave_total(q) / m + p.eps);
        if ((threadIdx.x & 63) == 0) {
            stat[g] = make_float2(mean, rstd);
            if (chunk == 0 && b.piece == 0) { p.mean[n * p.G + b.g_lo + g] = mean; p.rstd[n * p.G + b.g_lo + g] = rstd; }
        }
    }
    __syncthreads();
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int c0 = b.c_lo + lv * VEC;
    if (r >= p.P || c0 >= b.c_hi) return;
    GnStat<VEC, GS> st;
#pragma unroll
    for (int j = 0; j < (GS ? 1 : VEC); ++j) {
        const float2 t = stat[p.pieces == 1 ? (lv * VEC + j) / p.Cg : 0];
        st.m[j] = t.x; st.r[j] = t.y;
    }
    float ga[VEC], be[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { ga[j] = p.gamma[c0 + j] * st.rstd(j); be[j] = p.beta[c0 + j]; }
    const int s_hi = min(p.S, (chunk + 1) * p.chunk);
    with_act(p.act, [&](auto a) __attribute__((always_inline)) {
        for (int s0 = chunk * p.chunk + r; s0 < s_hi; s0 += U * p.P) {
            GnData<T, VEC> d[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s0 + u * p.P < s_hi) d[u].load(p.x, n * p.xn + (s0 + u * p.P) * p.xs + c0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * p.P;
                if (s < s_hi) {
                    float f[VEC];
                    d[u].get(f);
                    if constexpr (VEC * sizeof(T) == 16) { if (p.qo) ck_store<VEC>(p, f, n * p.S + s, c0); }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] = fmaf(f[j] - st.mean(j), ga[j], be[j]);
                    act_apply<T, decltype(a)::value>(f);
                    typename VecOf<T, VEC>::raw o;
                    vec_put(o, f);
                    *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
                }
            }
        }
    });
}

// dbeta[c], dgamma[c] = sums over the rows of part [rows][C]: 8 channels (64 bytes of a row) a block, 64 rows at a time
__global__ __launch_bounds__(512) void gn_param_grad_kernel(const float2* __restrict__ part, long long rows, int C, float* dgamma, float* dbeta) {
    __shared__ float2 red[64][8];
    const int c = blockIdx.x * 8 + (threadIdx.x & 7), k = threadIdx.x >> 3;
    float2 s = make_float2(0.f, 0.f);
    if (c < C)
#pragma unroll 4
        for (long long i = k; i < rows; i += 64) {
            const float2 t = part[i * C + c];
            s.x += t.x; s.y += t.y;
        }
    red[k][threadIdx.x & 7] = s;
    __syncthreads();
    if (threadIdx.x < 8 && c < C) {
        float2 t = make_float2(0.f, 0.f);
        for (int i = 0; i < 64; ++i) { t.x += red[i][threadIdx.x].x; t.y += red[i][threadIdx.x].y; }
        if (dbeta) dbeta[c] = t.x;
        if (dgamma) dgamma[c] = t.y;
    }
}

// ---- geometry ------------------------------------------------------------------------------------------------------------

GnPlan gn_plan(GnP& p, int es, int vec_max, bool backward, bool ckpt = false) {
    GnPlan pl;
    const int GT = backward ? GTB : GTF;
    // widest vector whose whole-group blocks (or pieces of one group) start on vector borders
    int vec = vec_max;
    for (;; vec = vec > 2 ? 2 : 1) {
        const long long unit = std::lcm((long long)p.Cg, (long long)vec);
        if (vec == 1 || unit <= (long long)GT * vec || p.Cg % vec == 0) break;
    }
    pl.vec = vec;
    pl.gs = p.Cg % vec == 0;
    const long long unit = std::lcm((long long)p.Cg, (long long)vec);
    const int cap = GT * vec;
    if (unit > cap) {                                       // a group wider than a workgroup's lanes
        p.CB = cap;
        p.pieces = cdiv(p.Cg, cap);
        p.ncb = p.G * p.pieces;
    } else {
        // at least 128 bytes of a position side by side (a cache line), and enough channels for every thread where S is short
        const long long want = std::max<long long>(128 / es, (long long)GT * vec / std::max(1, p.S));
        long long cb = unit;
        while (cb * 2 <= cap && cb < want && cb < p.C) cb *= 2;
        p.CB = (int)std::min<long long>(cb, p.C);
        p.pieces = 1;
        p.ncb = cdiv(p.C, p.CB);
    }
    const auto lanes = [&]() {
        p.LV = cdiv(p.CB, vec);
        p.P = GT / p.LV;
        p.NSUB = 1;
        if (p.P > p.S) { p.P = std::max(1, p.S); p.NSUB = std::min(GT / (p.LV * p.P), std::max(1, p.N)); }
        p.shuf = p.NSUB == 1 && p.LV <= 32 && (p.LV & (p.LV - 1)) == 0 && p.P * p.LV == GT;
    };
    lanes();
    // fewer channels side by side, down to 32 bytes, where a run of groups does not fit a workgroup's registers or where there would be
    // fewer workgroups than CUs (the blocks that share a cache line run on one XCD)
    while (p.pieces == 1 && p.CB % 2 == 0 && (p.CB / 2) % unit == 0 && p.CB / 2 * es >= 32 && !(ckpt && p.CB % 64) &&
           (cdiv(p.S, p.P) > ITEMS_MAX || (p.S * (long long)p.CB > 16 * vec * 64 && cdivll(p.N, p.NSUB) * p.ncb < 512))) {
        p.CB /= 2;
        p.ncb = cdiv(p.C, p.CB);
        lanes();
    }
    const long long held_blocks = cdivll(p.N, p.NSUB) * p.ncb;
    pl.held = p.pieces == 1 && cdiv(p.S, p.P) <= ITEMS_MAX && (held_blocks >= 64 || cdiv(p.S, p.P) <= 4);
    if (pl.held) {
        p.chunk = std::max(1, p.S);
        p.nchunk = 1;
        const int items = cdiv(p.S, p.P);
        pl.items = items;
        // backward: a workgroup goes over several samples and leaves one row of column sums
        pl.blocks = backward ? std::min<long long>(cdivll(p.N, p.NSUB), std::max(1, 2048 / p.ncb)) * p.ncb : held_blocks;
        pl.part = backward ? (size_t)(pl.blocks / p.ncb) * p.C : 0;
    } else {
        while (p.pieces == 1 && p.CB * es < 128 && p.CB * 2 <= std::min(cap, p.C)) p.CB *= 2;   // whole cache lines again
        if (p.pieces == 1) { p.ncb = cdiv(p.C, p.CB); p.LV = cdiv(p.CB, vec); }
        p.NSUB = 1;
        p.P = std::max(1, GT / p.LV);
        p.shuf = p.LV <= 32 && (p.LV & (p.LV - 1)) == 0 && p.P * p.LV == GT;
        pl.items = ITEMS_MAX;
        // forward: chunks of what a workgroup holds, shorter where that leaves the chip empty; backward: about 4096 workgroups
        long long chunk = backward ? cdivll(cdivll((long long)p.N * p.ncb * p.S, 4096), 4 * p.P) * 4 * p.P : (long long)p.P * ITEMS_MAX;
        while (chunk > 4 * p.P && (long long)p.N * p.ncb * cdivll(p.S, chunk) < 512) chunk = cdivll(chunk / 2, p.P) * p.P;
        p.chunk = (int)std::min<long long>(chunk, std::max(1, p.S));
        p.nchunk = std::max(1, cdiv(p.S, p.chunk));
        pl.blocks = (long long)p.N * p.ncb * p.nchunk;
        pl.part = backward ? (size_t)p.N * p.nchunk * p.C : (size_t)p.N * p.G * p.nchunk * p.pieces;
    }
    p.blocks = pl.blocks;
    return pl;
}

bool mult(long long a, int m) { return a % m == 0; }
int vec_of(const GnP& p, int es, bool backward) {
    // the widest vector that every pointer and stride allows
    for (int v : {16 / es, 2}) {
        bool ok = mult(p.C, v);
        const auto t = [&](const void* a, long long n, long long s) {
            ok = ok && (uintptr_t)a % (size_t)(v * es) == 0 && mult(n, v) && mult(s, v);
        };
        if (p.x) t(p.x, p.xn, p.xs);
        if (backward) t(p.dy, p.dn, p.ds);
        if (p.q) ok = ok && (uintptr_t)p.q % (size_t)v == 0;
        t(p.y, p.yn, p.ys);
        if (ok) return v;
    }
    return 1;
}

template <class T, int VEC, bool GS> int gn_fwd_t(const GnP& p, const GnPlan& pl, hipStream_t st) {
    const size_t lds = sizeof(float) * ((size_t)GTF * (GS ? 1 : VEC) + (size_t)p.NSUB * cdiv(p.CB, std::min(p.Cg, p.CB)));
    if (pl.held)
        return pl.items <= 4 ? gn_launch(gn_fwd_kernel<T, VEC, 4, GS, false>, p, GTF, lds, st) : gn_launch(gn_fwd_kernel<T, VEC, ITEMS_MAX, GS, false>, p, GTF, lds, st);
    const int rc = gn_launch(gn_fwd_kernel<T, VEC, ITEMS_MAX, GS, true>, p, GTF, lds, st);
    if (rc != FAVAE_OK) return rc;
    return gn_launch(gn_apply_kernel<T, VEC, GS>, p, GTF, sizeof(float2) * cdiv(p.CB, std::min(p.Cg, p.CB)), st);
}
template <class T> int gn_fwd(const GnP& p, const GnPlan& pl, hipStream_t st) {
#define GN_F(T_, V) { if constexpr (V == 1) return gn_fwd_t<T_, V, true>(p, pl, st); else return pl.gs ? gn_fwd_t<T_, V, true>(p, pl, st) : gn_fwd_t<T_, V, false>(p, pl, st); }
    GN_VEC(T, pl.vec, GN_F);
#undef GN_F
}
int gn_sizes(const char* who, long long N, long long S, int C, int G, int act, int dtype) {
    FAVAE_CHECK_ARG(dtype == FAVAE_F32 || dtype == FAVAE_BF16, "%s: dtype is neither fp32 nor bf16", who);
    FAVAE_CHECK_ARG(act >= FAVAE_ACT_NONE && act <= FAVAE_ACT_GELU_TANH, "%s: unknown activation %d", who, act);
    FAVAE_CHECK_ARG(N >= 0 && S >= 0 && C >= 1 && G >= 1 && C % G == 0, "%s: C = %d channels do not divide into G = %d groups, or a negative size", who, C, G);
    FAVAE_CHECK_ARG(N <= 0x7fffffff && S <= 0x3fffffff && C <= (1 << 24), "%s: N, S or C too large", who);
    return FAVAE_OK;
}

}  // namespace

extern "C" size_t favae_gn_act_scratch(long long N, long long S, int C, int G, int backward, int dtype) {
    if (gn_sizes("favae_gn_act_scratch", N, S, C, G, FAVAE_ACT_NONE, dtype) != FAVAE_OK) return 0;
    // the plan depends on the vector width, which alignment decides: the largest over the widths
    size_t need = 0;
    for (int v : {dtype == FAVAE_F32 ? 4 : 8, 2, 1}) {
        if (C % v) continue;
        GnP p = {};
        p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G;
        for (bool ckpt : {false, true}) {
            GnP t = p;
            need = std::max(need, gn_plan(t, dtype == FAVAE_F32 ? 4 : 2, v, backward != 0, ckpt).part);
        }
    }
    return need * sizeof(float2);
}

extern "C" int favae_gn_act_fwd(const void* x, long long xn, long long xs, long long N, long long S, int C, int G, const float* gamma,
                                const float* beta, float eps, int act, void* y, long long yn, long long ys, float* mean, float* rstd,
                                void* q, void* e, void* scratch, size_t scratch_bytes, int dtype, void* stream) {
    const int rc = gn_sizes("favae_gn_act_fwd", N, S, C, G, act, dtype);
    if (rc != FAVAE_OK) return rc;
    if (N == 0) return FAVAE_OK;
    FAVAE_CHECK_ARG(gamma && beta && mean && rstd && (S == 0 || (x && y)), "favae_gn_act_fwd: null pointer");
    FAVAE_CHECK_ARG((q != nullptr) == (e != nullptr), "favae_gn_act_fwd: q and e, or neither");
    FAVAE_CHECK_ARG(S <= 1 || (xs >= C && ys >= C), "favae_gn_act_fwd: a position's stride is below C");
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    GnP p = {};
    p.x = x; p.xn = xn; p.xs = xs; p.y = y; p.yn = yn; p.ys = ys;
    p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd; p.part = (float2*)scratch;
    p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G; p.act = act; p.eps = eps;
    const GnPlan pl = gn_plan(p, es, vec_of(p, es, false), false, q != nullptr);
    FAVAE_CHECK_ARG(pl.part * sizeof(float2) <= scratch_bytes && (pl.part == 0 || scratch), "favae_gn_act_fwd: scratch of %zu bytes, %zu needed", scratch_bytes,
                    pl.part * sizeof(float2));
    if (q && S > 0) {
        p.nb = cdiv(C, CK_BLOCK);
        // the checkpoint leaves with y where the lanes of a wave hold whole blocks of 32 channels; otherwise a launch of its own first
        if (pl.vec * es == 16 && C % CK_BLOCK == 0 && p.CB % CK_BLOCK == 0 && ((uintptr_t)q & 7) == 0) {
            p.qo = (unsigned char*)q;
            p.eo = (unsigned char*)e;
        } else {
            FAVAE_CHECK_ARG(N == 1 || S == 1 || xn == S * xs, "favae_gn_act_fwd: a checkpoint of x needs one stride between all its rows");
            const int r2 = favae_ckpt8_pack(x, S == 1 ? xn : xs, N * S, C, q, C, e, p.nb, dtype, stream);
            if (r2 != FAVAE_OK) return r2;
        }
    }
    return dtype == FAVAE_F32 ? gn_fwd<float>(p, pl, (hipStream_t)stream) : gn_fwd<bf16_t>(p, pl, (hipStream_t)stream);
}

extern "C" int favae_gn_act_bwd(const void* dy, long long dn, long long ds, const void* x, long long xn, long long xs, const void* q, const void* e,
                                long long N, long long S, int C, int G, const float* gamma, const float* beta, const float* mean,
                                const float* rstd, int act, void* dx, long long dxn, long long dxs, float* dgamma, float* dbeta,
                                void* scratch, size_t scratch_bytes, int dtype, void* stream) {
    const int rc = gn_sizes("favae_gn_act_bwd", N, S, C, G, act, dtype);
    if (rc != FAVAE_OK) return rc;
    FAVAE_CHECK_ARG(gamma && beta && (N == 0 || S == 0 || (dy && dx && mean && rstd)), "favae_gn_act_bwd: null pointer");
    FAVAE_CHECK_ARG(N == 0 || S == 0 || (x != nullptr) != (q != nullptr && e != nullptr), "favae_gn_act_bwd: x, or its 8-bit checkpoint (q and e), and not both");
    FAVAE_CHECK_ARG(S <= 1 || (ds >= C && dxs >= C && (!x || xs >= C)), "favae_gn_act_bwd: a position's stride is below C");
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    const hipStream_t st = (hipStream_t)stream;
    GnP p = {};
    p.x = x; p.xn = xn; p.xs = xs; p.q = (const unsigned char*)q; p.e = (const unsigned char*)e; p.dy = dy; p.dn = dn; p.ds = ds;
    p.y = dx; p.yn = dxn; p.ys = dxs;
    p.gamma = gamma; p.beta = beta; p.mean = (float*)mean; p.rstd = (float*)rstd; p.part = (float2*)scratch;
    p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G; p.act = act; p.nb = cdiv(C, CK_BLOCK);
    long long rows = 0;
    if (N > 0 && S > 0) {
        const GnPlan pl = gn_plan(p, es, vec_of(p, es, true), true);
        FAVAE_CHECK_ARG(pl.part * sizeof(float2) <= scratch_bytes && scratch, "favae_gn_act_bwd: scratch of %zu bytes, %zu needed", scratch_bytes,
                        pl.part * sizeof(float2));
        rows = (long long)(pl.part / C);
        const int r2 = dtype == FAVAE_F32 ? gn_bwd_f32(p, pl, st) : gn_bwd_bf16(p, pl, st);
        if (r2 != FAVAE_OK) return r2;
    }
    if (dgamma || dbeta) {
        gn_param_grad_kernel<<<cdiv(C, 8), 512, 0, st>>>((const float2*)scratch, rows, C, dgamma, dbeta);
        FAVAE_LAUNCH_CHECK();
    }
    return FAVAE_OK;
}
