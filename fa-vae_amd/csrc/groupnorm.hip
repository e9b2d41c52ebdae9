// Group norm with an activation over channels-last maps, forward and backward.
//
//   per sample n and group g, over the m = S * Cg values of its S positions and Cg channels:
//     mean = sum x / m,  rstd = (sum (x - mean)^2 / m + eps)^-1/2,  xh = (x - mean) rstd,  z = gamma xh + beta,  y = act(z)
//   backward:  dz = dy act'(z),  dbeta = sum dz,  dgamma = sum dz xh  (over samples and positions),
//     dx = rstd (gamma dz - (s1 + xh s2) / m),  s1 = sum over the group of gamma dz,  s2 = sum over the group of gamma dz xh
//
// Memory bounds both.  Held form: one workgroup holds all positions of a run of whole groups in registers, so that the input is read
// once: load, sum, sum of squared distances from the mean (no cancellation), normalise, store.  Chunked form, where a group is too
// large for one workgroup's registers or there are too few groups to fill the chip: a first launch leaves the partial sums of each
// chunk of positions, a second one joins them and makes the pass over the data.  Sums are fp32 within a chunk and joined in a fixed
// order: the results do not depend on scheduling.
#include "act8.h"
#include <algorithm>
#include <numeric>

namespace {

constexpr int GT = 512;                 // threads of a workgroup

struct GnP {
    const void *x, *dy;
    void* y;                            // y, or dx
    const unsigned char *q, *e;         // x as an 8-bit checkpoint, [N][S][C] and [N][S][nb]
    long long xn, xs, dn, ds, yn, ys;   // strides of a sample and of a position, in elements
    const float *gamma, *beta;
    float *mean, *rstd;                 // [N][G]
    float2* part;                       // partial sums, see the kernels
    int N, S, C, G, Cg, act, nb;
    float eps;
    // geometry.  A workgroup takes CB channels: whole groups (pieces == 1), or piece j of `pieces` of one group wider than it.
    // LV lanes side by side cover the CB channels, P rows of lanes take P positions at once, NSUB samples share a workgroup.
    int LV, P, NSUB, CB, ncb, pieces, chunk, nchunk, shuf;
    long long blocks;
};

struct GnBlock { int c_lo, c_hi, g_lo, ng, cw, piece; };   // channels, groups, channels of a group inside this block
__device__ __forceinline__ GnBlock gn_block(const GnP& p, int cb) {
    GnBlock b;
    if (p.pieces == 1) {
        b.c_lo = cb * p.CB; b.c_hi = min(p.C, b.c_lo + p.CB);
        b.g_lo = b.c_lo / p.Cg; b.ng = (b.c_hi - b.c_lo) / p.Cg; b.cw = p.Cg; b.piece = 0;
    } else {
        b.g_lo = cb / p.pieces; b.piece = cb - b.g_lo * p.pieces; b.ng = 1;
        b.c_lo = b.g_lo * p.Cg + b.piece * p.CB; b.c_hi = min((b.g_lo + 1) * p.Cg, b.c_lo + p.CB);
        b.cw = b.c_hi - b.c_lo;
    }
    return b;
}
// consecutive logical blocks (the channel blocks of one sample read the same cache lines) go to one XCD: the launch deals blocks to
// the 8 XCDs in turn
__device__ __forceinline__ long long xcd_order(long long b, long long n) {
    const long long per = n / 8;
    return b < per * 8 ? (b & 7) * per + (b >> 3) : b;
}

__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Sum of v over the threads of every (sample of the block, group of the block) pair into grp[].  A thread's NV values belong to
// columns lv * NV + j of its row; a group is cpg neighbouring columns.  With p.shuf the 64 / LV rows of a wave are added by
// shuffles first.  Every thread of the block calls; values of idle threads are 0.
template <int NV>
__device__ __forceinline__ void gn_reduce(const GnP& p, float (&v)[NV], float* red, float* grp, int lv, int r, int ng, int cpg) {
    const int cols = p.LV * NV;
    int rows = p.P;
    if (p.shuf) {
        for (int o = p.LV; o < 64; o <<= 1)
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] += __shfl_xor(v[j], o, 64);
        rows = GT / 64;
        if ((int)(threadIdx.x & 63) < p.LV)
#pragma unroll
            for (int j = 0; j < NV; ++j) red[(threadIdx.x >> 6) * cols + lv * NV + j] = v[j];
    } else if (r < p.P * p.NSUB) {
#pragma unroll
        for (int j = 0; j < NV; ++j) red[r * cols + lv * NV + j] = v[j];
    }
    __syncthreads();
    const int pairs = p.NSUB * ng, per = rows * cpg;
    if (per <= 32 || pairs >= GT) {
        for (int k = threadIdx.x; k < pairs; k += GT) {
            const int sub = k / ng, g = k - sub * ng;
            float s = 0.f;
            for (int i = 0; i < rows; ++i)
                for (int c = 0; c < cpg; ++c) s += red[(sub * rows + i) * cols + g * cpg + c];
            grp[k] = s;
        }
    } else {
        for (int k = threadIdx.x >> 6; k < pairs; k += GT / 64) {
            const int sub = k / ng, g = k - sub * ng;
            float s = 0.f;
            for (int i = threadIdx.x & 63; i < per; i += 64) {
                const int row = i / cpg, c = i - row * cpg;
                s += red[(sub * rows + row) * cols + g * cpg + c];
            }
            s = wave_total(s);
            if ((threadIdx.x & 63) == 0) grp[k] = s;
        }
    }
    __syncthreads();
}

template <class T, int VEC> struct GnData {
    typedef typename VecOf<T, VEC>::raw raw;
    raw v;
    __device__ __forceinline__ void load(const void* base, long long off) { v = *(const raw*)((const T*)base + off); }
    __device__ __forceinline__ void get(float (&f)[VEC]) const { vec_get(f, v); }
};
// VEC values of an 8-bit checkpoint: they lie inside one block of 32 (VEC divides 32 and their first channel)
template <int VEC> struct CkData {
    unsigned w[VEC == 8 ? 2 : 1];
    float s;
    __device__ __forceinline__ void load(const unsigned char* q, const unsigned char* e, long long pos, int C, int nb, int c) {
        const unsigned char* a = q + pos * C + c;
        if constexpr (VEC == 8) { const uint2 t = *(const uint2*)a; w[0] = t.x; w[1] = t.y; }
        else if constexpr (VEC == 4) w[0] = *(const unsigned*)a;
        else if constexpr (VEC == 2) w[0] = *(const unsigned short*)a;
        else w[0] = *a;
        s = ck_scale(e[pos * nb + (c >> 5)]);
    }
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = ck_value(w[j >> 2], j & 3, s);
    }
};

// Per-channel constants of a thread.  GS: a vector lies inside one group, so that its mean and rstd are single values.
template <int VEC, bool GS> struct GnStat {
    float m[GS ? 1 : VEC], r[GS ? 1 : VEC];
    __device__ __forceinline__ float mean(int j) const { return m[GS ? 0 : j]; }
    __device__ __forceinline__ float rstd(int j) const { return r[GS ? 0 : j]; }
};

// ---- forward -------------------------------------------------------------------------------------------------------------
// STATS: leave (mean, sum of squared distances) of this chunk in part[((n G + g) nchunk + chunk) pieces + piece] and stop.
template <class T, int VEC, int ITEMS, bool GS, bool STATS> __global__ __launch_bounds__(GT) void gn_fwd_kernel(const GnP p) {
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
    float* grp = lds + GT * NV;

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
    if ((int)threadIdx.x < pairs && pairs <= GT) keep_mean = grp[threadIdx.x] * inv;
    if (pairs > GT)                              // more pairs than threads: through memory at once (grp is reused below)
        for (int k = threadIdx.x; k < pairs; k += GT) {
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
        }
    }
    gn_reduce<NV>(p, v, red, grp, lv, r, b.ng, cpg);
    for (int k = threadIdx.x; k < pairs; k += GT) {
        const long long nn = nb0 * p.NSUB + k / b.ng;
        const int g = b.g_lo + k % b.ng;
        if (nn < p.N) {
            if constexpr (STATS) {
                float2* o = p.part + ((nn * p.G + g) * p.nchunk + chunk) * p.pieces + b.piece;
                if (pairs <= GT) o->x = keep_mean;
                o->y = grp[k];
            } else {
                if (pairs <= GT) p.mean[nn * p.G + g] = keep_mean;
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
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int s = s_lo + pos + i * p.P;
            if (s < s_hi) {
                float f[VEC];
                d[i].get(f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[j] = fmaf(f[j] - st.mean(j), ga[j], be[j]);
                act_apply<T>(f, p.act);
                typename VecOf<T, VEC>::raw o;
                vec_put(o, f);
                *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
            }
        }
    }
}

// Chunked form, second launch: join the chunks of this block's groups (mean of means, and sums of squared distances moved to it), normalise.
template <class T, int VEC, bool GS> __global__ __launch_bounds__(GT) void gn_apply_kernel(const GnP p) {
    extern __shared__ float lds[];
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const int chunk = (int)(t_ % p.nchunk);
    const long long n = t_ / p.nchunk;
    const GnBlock b = gn_block(p, cb);
    const int parts = p.nchunk * p.pieces;
    float2* stat = (float2*)lds;                 // [ng] (mean, rstd)
    for (int g = threadIdx.x >> 6; g < b.ng; g += GT / 64) {
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
#pragma unroll 4
    for (int s = chunk * p.chunk + r; s < s_hi; s += p.P) {
        GnData<T, VEC> d;
        d.load(p.x, n * p.xn + s * p.xs + c0);
        float f[VEC];
        d.get(f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = fmaf(f[j] - st.mean(j), ga[j], be[j]);
        act_apply<T>(f, p.act);
        typename VecOf<T, VEC>::raw o;
        vec_put(o, f);
        *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------------
// Column sums (dz, dz xh) of a block's threads into tot[sub][CB] (float2).  red: [rows][CB] float2.
template <int VEC>
__device__ __forceinline__ void gn_columns(const GnP& p, float (&a)[VEC], float (&bq)[VEC], float2* red, float2* tot, int lv, int r) {
    const int cols = p.LV * VEC;
    int rows = p.P;
    if (p.shuf) {
        for (int o = p.LV; o < 64; o <<= 1)
#pragma unroll
            for (int j = 0; j < VEC; ++j) { a[j] += __shfl_xor(a[j], o, 64); bq[j] += __shfl_xor(bq[j], o, 64); }
        rows = GT / 64;
        if ((int)(threadIdx.x & 63) < p.LV)
#pragma unroll
            for (int j = 0; j < VEC; ++j) red[(threadIdx.x >> 6) * cols + lv * VEC + j] = make_float2(a[j], bq[j]);
    } else if (r < p.P * p.NSUB) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) red[r * cols + lv * VEC + j] = make_float2(a[j], bq[j]);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < p.NSUB * cols; k += GT) {
        const int sub = k / cols, c = k - sub * cols;
        float2 s = make_float2(0.f, 0.f);
        for (int i = 0; i < rows; ++i) {
            const float2 t = red[(sub * rows + i) * cols + c];
            s.x += t.x; s.y += t.y;
        }
        tot[k] = s;
    }
    __syncthreads();
}

// SUMS: leave the column sums of the chunk in part[(n nchunk + chunk) C + c] and stop.  Otherwise the block takes samples blockIdx,
// + gridDim, ...: dx, and its column sums over all of them in part[blockIdx C + c].
template <class T, int VEC, int ITEMS, bool GS, bool CK, bool SUMS> __global__ __launch_bounds__(GT) void gn_bwd_kernel(const GnP p) {
    extern __shared__ float lds[];
    const int cols = p.LV * VEC;
    float2* red = (float2*)lds;
    float2* tot = red + (p.shuf ? (GT / 64) * cols : p.P * p.NSUB * cols);
    float2* grp = tot + p.NSUB * cols;           // [NSUB][ng]
    float2* acc = grp + p.NSUB * cols;           // [cols] (held form)
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const int chunk = SUMS ? (int)(t_ % p.nchunk) : 0;
    const long long first = SUMS ? t_ / p.nchunk : t_;
    const long long stride = SUMS ? p.N : p.blocks / p.ncb;
    const GnBlock b = gn_block(p, cb);
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int sub = r / p.P, pos = r - sub * p.P;
    const int c0 = b.c_lo + lv * VEC;
    const int s_lo = chunk * p.chunk, s_hi = min(p.S, s_lo + p.chunk);
    const bool col_ok = sub < p.NSUB && c0 < b.c_hi;
    float ga[VEC], be[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { ga[j] = col_ok ? p.gamma[c0 + j] : 0.f; be[j] = col_ok ? p.beta[c0 + j] : 0.f; }
    if constexpr (!SUMS)
        for (int k = threadIdx.x; k < cols; k += GT) acc[k] = make_float2(0.f, 0.f);
    const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
    for (long long nb0 = first; nb0 * p.NSUB < p.N; nb0 += stride) {
        const long long n = nb0 * p.NSUB + sub;
        const bool active = col_ok && n < p.N;
        GnStat<VEC, GS> st;
#pragma unroll
        for (int j = 0; j < (GS ? 1 : VEC); ++j) {
            const int g = b.g_lo + (p.pieces == 1 ? (lv * VEC + j) / p.Cg : 0);
            st.m[j] = active ? p.mean[n * p.G + g] : 0.f;
            st.r[j] = active ? p.rstd[n * p.G + g] : 0.f;
        }
        GnData<T, VEC> d[ITEMS];
        typename std::conditional<CK, CkData<VEC>, GnData<T, VEC>>::type xv[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int s = s_lo + pos + i * p.P;
            if (active && s < s_hi) {
                if constexpr (CK) xv[i].load(p.q, p.e, n * p.S + s, p.C, p.nb, c0);
                else xv[i].load(p.x, n * p.xn + s * p.xs + c0);
                d[i].load(p.dy, n * p.dn + s * p.ds + c0);
            }
        }
        float sa[VEC], sb[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) sa[j] = sb[j] = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (active && s_lo + pos + i * p.P < s_hi) {
                float xh[VEC], z[VEC], g[VEC];
                xv[i].get(xh);
                d[i].get(g);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { xh[j] = (xh[j] - st.mean(j)) * st.rstd(j); z[j] = fmaf(xh[j], ga[j], be[j]); }
                act_grad_mul<T>(g, z, p.act);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { sa[j] += g[j]; sb[j] = fmaf(g[j], xh[j], sb[j]); }
            }
        }
        gn_columns<VEC>(p, sa, sb, red, tot, lv, r);
        if constexpr (SUMS) {
            for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += GT) p.part[(nb0 * p.nchunk + chunk) * p.C + b.c_lo + k] = tot[k];
        } else {
            for (int k = threadIdx.x; k < cols; k += GT) {
                float2 t = acc[k];
                for (int u = 0; u < p.NSUB; ++u) { t.x += tot[u * cols + k].x; t.y += tot[u * cols + k].y; }
                acc[k] = t;
            }
            const int pairs = p.NSUB * b.ng;
            if (b.cw <= 32 || pairs >= GT) {
                for (int k = threadIdx.x; k < pairs; k += GT) {
                    const int u = k / b.ng, g = k - u * b.ng;
                    float2 s = make_float2(0.f, 0.f);
                    for (int c = g * b.cw; c < (g + 1) * b.cw; ++c) {
                        const float2 t = tot[u * cols + c];
                        const float w = p.gamma[b.c_lo + c];
                        s.x = fmaf(w, t.x, s.x); s.y = fmaf(w, t.y, s.y);
                    }
                    grp[k] = s;
                }
            } else {
                for (int k = threadIdx.x >> 6; k < pairs; k += GT / 64) {
                    const int u = k / b.ng, g = k - u * b.ng;
                    float2 s = make_float2(0.f, 0.f);
                    for (int c = g * b.cw + (threadIdx.x & 63); c < (g + 1) * b.cw; c += 64) {
                        const float2 t = tot[u * cols + c];
                        const float w = p.gamma[b.c_lo + c];
                        s.x = fmaf(w, t.x, s.x); s.y = fmaf(w, t.y, s.y);
                    }
                    s.x = wave_total(s.x); s.y = wave_total(s.y);
                    if ((threadIdx.x & 63) == 0) grp[k] = s;
                }
            }
            __syncthreads();
            if (active) {
                GnStat<VEC, GS> gs;                  // (s1 / m, s2 / m) of the groups
#pragma unroll
                for (int j = 0; j < (GS ? 1 : VEC); ++j) {
                    const float2 t = grp[sub * b.ng + (lv * VEC + j) / p.Cg];
                    gs.m[j] = t.x * inv_m; gs.r[j] = t.y * inv_m;
                }
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const int s = s_lo + pos + i * p.P;
                    if (s < s_hi) {
                        float xh[VEC], z[VEC], g[VEC];
                        xv[i].get(xh);
                        d[i].get(g);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) { xh[j] = (xh[j] - st.mean(j)) * st.rstd(j); z[j] = fmaf(xh[j], ga[j], be[j]); }
                        act_grad_mul<T>(g, z, p.act);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) g[j] = st.rstd(j) * (fmaf(ga[j], g[j], -gs.mean(j)) - xh[j] * gs.rstd(j));
                        typename VecOf<T, VEC>::raw o;
                        vec_put(o, g);
                        *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
                    }
                }
            }
            __syncthreads();                          // red, tot and grp are free again
        }
    }
    if constexpr (!SUMS)
        for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += GT) p.part[first * p.C + b.c_lo + k] = acc[k];
}

// Chunked form, second launch: s1 and s2 of this block's groups from the column sums of every chunk, then dx.
template <class T, int VEC, bool GS, bool CK> __global__ __launch_bounds__(GT) void gn_bwd_apply_kernel(const GnP p) {
    extern __shared__ float lds[];
    float2* grp = (float2*)lds;
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const int chunk = (int)(t_ % p.nchunk);
    const long long n = t_ / p.nchunk;
    const GnBlock b = gn_block(p, cb);
    const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
    for (int g = threadIdx.x >> 6; g < b.ng; g += GT / 64) {
        float2 s = make_float2(0.f, 0.f);
        for (int i = threadIdx.x & 63; i < p.nchunk * p.Cg; i += 64) {
            const int ch = i / p.Cg, c = (b.g_lo + g) * p.Cg + (i - ch * p.Cg);
            const float2 t = p.part[(n * p.nchunk + ch) * p.C + c];
            const float w = p.gamma[c];
            s.x = fmaf(w, t.x, s.x); s.y = fmaf(w, t.y, s.y);
        }
        s.x = wave_total(s.x); s.y = wave_total(s.y);
        if ((threadIdx.x & 63) == 0) grp[g] = make_float2(s.x * inv_m, s.y * inv_m);
    }
    __syncthreads();
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int c0 = b.c_lo + lv * VEC;
    if (r >= p.P || c0 >= b.c_hi) return;
    GnStat<VEC, GS> st, gs;
#pragma unroll
    for (int j = 0; j < (GS ? 1 : VEC); ++j) {
        const int g = p.pieces == 1 ? (lv * VEC + j) / p.Cg : 0;
        st.m[j] = p.mean[n * p.G + b.g_lo + g];
        st.r[j] = p.rstd[n * p.G + b.g_lo + g];
        gs.m[j] = grp[g].x; gs.r[j] = grp[g].y;
    }
    float ga[VEC], be[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { ga[j] = p.gamma[c0 + j]; be[j] = p.beta[c0 + j]; }
    const int s_hi = min(p.S, (chunk + 1) * p.chunk);
#pragma unroll 2
    for (int s = chunk * p.chunk + r; s < s_hi; s += p.P) {
        typename std::conditional<CK, CkData<VEC>, GnData<T, VEC>>::type xv;
        GnData<T, VEC> d;
        if constexpr (CK) xv.load(p.q, p.e, n * p.S + s, p.C, p.nb, c0);
        else xv.load(p.x, n * p.xn + s * p.xs + c0);
        d.load(p.dy, n * p.dn + s * p.ds + c0);
        float xh[VEC], z[VEC], g[VEC];
        xv.get(xh);
        d.get(g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) { xh[j] = (xh[j] - st.mean(j)) * st.rstd(j); z[j] = fmaf(xh[j], ga[j], be[j]); }
        act_grad_mul<T>(g, z, p.act);
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = st.rstd(j) * (fmaf(ga[j], g[j], -gs.mean(j)) - xh[j] * gs.rstd(j));
        typename VecOf<T, VEC>::raw o;
        vec_put(o, g);
        *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
    }
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
constexpr int ITEMS_MAX = 16;
struct GnPlan { int vec; bool gs, held; int items; long long blocks; size_t part; };   // part: float2 entries of workspace

GnPlan gn_plan(GnP& p, int es, int vec_max, bool backward) {
    GnPlan pl;
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
    // a run of groups that does not fit a workgroup's registers may fit with fewer channels side by side (the blocks that share its
    // cache lines run on one XCD): down to 32 bytes
    while (p.pieces == 1 && cdiv(p.S, p.P) > ITEMS_MAX && p.CB % 2 == 0 && (p.CB / 2) % unit == 0 && p.CB / 2 * es >= 32) {
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
        pl.items = items <= 4 ? 4 : ITEMS_MAX;
        // backward: a workgroup goes over several samples and leaves one row of column sums
        pl.blocks = backward ? std::min<long long>(cdivll(p.N, p.NSUB), std::max(1, 2048 / p.ncb)) * p.ncb : held_blocks;
        pl.part = backward ? (size_t)(pl.blocks / p.ncb) * p.C : 0;
    } else {
        p.NSUB = 1;
        p.P = std::max(1, GT / p.LV);
        p.shuf = p.LV <= 32 && (p.LV & (p.LV - 1)) == 0 && p.P * p.LV == GT;
        pl.items = ITEMS_MAX;
        // chunks of what a workgroup holds, shorter where that leaves the chip empty
        long long chunk = (long long)p.P * ITEMS_MAX;
        while (chunk > 4 * p.P && (long long)p.N * p.ncb * cdivll(p.S, chunk) < 512) chunk /= 2;
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

#define GN_VEC(T, vec, F)                                                              \
    do {                                                                               \
        if constexpr (sizeof(T) == 4) { if ((vec) == 4) F(T, 4) else if ((vec) == 2) F(T, 2) else F(T, 1) } \
        else { if ((vec) == 8) F(T, 8) else if ((vec) == 2) F(T, 2) else F(T, 1) }     \
    } while (0)

template <class K> int gn_launch(K k, const GnP& p, size_t lds, hipStream_t st) {
    FAVAE_CHECK_ARG(p.blocks <= 0x7fffffffLL, "favae_gn_act: too many samples for one launch");
    if (p.blocks > 0) k<<<(unsigned)p.blocks, GT, lds, st>>>(p);
    FAVAE_LAUNCH_CHECK();
    return FAVAE_OK;
}

template <class T, int VEC, bool GS> int gn_fwd_t(const GnP& p, const GnPlan& pl, hipStream_t st) {
    const size_t lds = sizeof(float) * ((size_t)GT * (GS ? 1 : VEC) + (size_t)p.NSUB * cdiv(p.CB, std::min(p.Cg, p.CB)));
    if (pl.held)
        return pl.items == 4 ? gn_launch(gn_fwd_kernel<T, VEC, 4, GS, false>, p, lds, st) : gn_launch(gn_fwd_kernel<T, VEC, ITEMS_MAX, GS, false>, p, lds, st);
    const int rc = gn_launch(gn_fwd_kernel<T, VEC, ITEMS_MAX, GS, true>, p, lds, st);
    if (rc != FAVAE_OK) return rc;
    return gn_launch(gn_apply_kernel<T, VEC, GS>, p, sizeof(float2) * cdiv(p.CB, std::min(p.Cg, p.CB)), st);
}
template <class T, int VEC, bool GS, bool CK> int gn_bwd_t(const GnP& p, const GnPlan& pl, hipStream_t st) {
    const int cols = p.LV * VEC;
    const size_t lds = sizeof(float2) * ((size_t)(p.shuf ? GT / 64 : p.P * p.NSUB) * cols + 2 * (size_t)p.NSUB * cols + cols);
    if (pl.held)
        return pl.items == 4 ? gn_launch(gn_bwd_kernel<T, VEC, 4, GS, CK, false>, p, lds, st)
                             : gn_launch(gn_bwd_kernel<T, VEC, ITEMS_MAX, GS, CK, false>, p, lds, st);
    const int rc = gn_launch(gn_bwd_kernel<T, VEC, ITEMS_MAX, GS, CK, true>, p, lds, st);
    if (rc != FAVAE_OK) return rc;
    return gn_launch(gn_bwd_apply_kernel<T, VEC, GS, CK>, p, sizeof(float2) * cdiv(p.CB, std::min(p.Cg, p.CB)), st);
}
template <class T> int gn_fwd(const GnP& p, const GnPlan& pl, hipStream_t st) {
#define GN_F(T_, V) { return pl.gs ? gn_fwd_t<T_, V, true>(p, pl, st) : gn_fwd_t<T_, V, false>(p, pl, st); }
    GN_VEC(T, pl.vec, GN_F);
#undef GN_F
}
template <class T, bool CK> int gn_bwd(const GnP& p, const GnPlan& pl, hipStream_t st) {
#define GN_F(T_, V) { return pl.gs ? gn_bwd_t<T_, V, true, CK>(p, pl, st) : gn_bwd_t<T_, V, false, CK>(p, pl, st); }
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
        need = std::max(need, gn_plan(p, dtype == FAVAE_F32 ? 4 : 2, v, backward != 0).part);
    }
    return need * sizeof(float2);
}

extern "C" int favae_gn_act_fwd(const void* x, long long xn, long long xs, long long N, long long S, int C, int G, const float* gamma,
                                const float* beta, float eps, int act, void* y, long long yn, long long ys, float* mean, float* rstd,
                                void* scratch, size_t scratch_bytes, int dtype, void* stream) {
    const int rc = gn_sizes("favae_gn_act_fwd", N, S, C, G, act, dtype);
    if (rc != FAVAE_OK) return rc;
    if (N == 0) return FAVAE_OK;
    FAVAE_CHECK_ARG(gamma && beta && mean && rstd && (S == 0 || (x && y)), "favae_gn_act_fwd: null pointer");
    FAVAE_CHECK_ARG(S <= 1 || (xs >= C && ys >= C), "favae_gn_act_fwd: a position's stride is below C");
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    GnP p = {};
    p.x = x; p.xn = xn; p.xs = xs; p.y = y; p.yn = yn; p.ys = ys;
    p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd; p.part = (float2*)scratch;
    p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G; p.act = act; p.eps = eps;
    const GnPlan pl = gn_plan(p, es, vec_of(p, es, false), false);
    FAVAE_CHECK_ARG(pl.part * sizeof(float2) <= scratch_bytes && (pl.part == 0 || scratch), "favae_gn_act_fwd: scratch of %zu bytes, %zu needed", scratch_bytes,
                    pl.part * sizeof(float2));
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
        const int r2 = dtype == FAVAE_F32 ? (q ? gn_bwd<float, true>(p, pl, st) : gn_bwd<float, false>(p, pl, st))
                                          : (q ? gn_bwd<bf16_t, true>(p, pl, st) : gn_bwd<bf16_t, false>(p, pl, st));
        if (r2 != FAVAE_OK) return r2;
    }
    if (dgamma || dbeta) {
        gn_param_grad_kernel<<<cdiv(C, 8), 512, 0, st>>>((const float2*)scratch, rows, C, dgamma, dbeta);
        FAVAE_LAUNCH_CHECK();
    }
    return FAVAE_OK;
}
