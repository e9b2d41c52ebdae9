// Backward kernels of group norm with an activation (formulas and the two forms: groupnorm.hip).
#pragma once
#include "groupnorm.h"

namespace {


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
        rows = GTB / 64;
        if ((int)(threadIdx.x & 63) < p.LV)
#pragma unroll
            for (int j = 0; j < VEC; ++j) red[(threadIdx.x >> 6) * cols + lv * VEC + j] = make_float2(a[j], bq[j]);
    } else if (r < p.P * p.NSUB) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) red[r * cols + lv * VEC + j] = make_float2(a[j], bq[j]);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < p.NSUB * cols; k += GTB) {
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

// Held form: the block takes samples blockIdx, + gridDim, ...: dx, and its column sums over all of them in part[blockIdx C + c].
// ACT: the activation, or -1: p.act (a choice inside the kernel costs the wide form its last registers).
// Lanes without a channel, a sample or a position read the last valid one instead and count for nothing, so that only stores are
// under a lane mask.  Items are kept one after the other: interleaved by the compiler they would need the registers of all at once.
template <class T, int VEC, int ITEMS, bool GS, bool CK, int ACT> __global__ __launch_bounds__(GTB) void gn_bwd_kernel(const GnP p) {
    extern __shared__ float lds[];
    const int cols = p.LV * VEC;
    float2* red = (float2*)lds;
    float2* tot = red + (p.shuf ? (GTB / 64) * cols : p.P * p.NSUB * cols);
    float2* grp = tot + p.NSUB * cols;           // [NSUB][ng]
    float2* acc = grp + p.NSUB * cols;           // [cols] (held form)
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const long long first = t_, stride = p.blocks / p.ncb;
    const GnBlock b = gn_block(p, cb);
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int sub = r / p.P;
    int pos = r - sub * p.P;
    const int last = p.S - 1;
    const bool col_ok = sub < p.NSUB && b.c_lo + lv * VEC < b.c_hi;
    const int c0 = min(b.c_lo + lv * VEC, b.c_hi - VEC);
    const int gl = (c0 - b.c_lo) / p.Cg;
    for (int k = threadIdx.x; k < cols; k += GTB) acc[k] = make_float2(0.f, 0.f);
    const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
    for (long long nb0 = first; nb0 * p.NSUB < p.N; nb0 += stride) {
        const long long n0 = nb0 * p.NSUB + sub, n = min(n0, (long long)p.N - 1);
        const bool active = col_ok && n0 < p.N;
        asm volatile("" : "+v"(pos));            // the items' offsets are made where they are used, not kept over the samples
        GnData<T, VEC> d[ITEMS];
        typename std::conditional<CK, CkData<VEC>, GnData<T, VEC>>::type xv[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int s = min(pos + i * p.P, last);
            if constexpr (CK) xv[i].load(p.q, p.e, n * p.S + s, p.C, p.nb, c0);
            else xv[i].load(p.x, n * p.xn + s * p.xs + c0);
            d[i].load(p.dy, n * p.dn + s * p.ds + c0);
        }
        GnStat<VEC, GS> st;
        float a[VEC];                                // gamma rstd
        float dz[ITEMS][VEC];             // held: its exp and reciprocal are half the work of a pass
        {
            float be[VEC], sa[VEC], sb[VEC];
#pragma unroll
            for (int j = 0; j < (GS ? 1 : VEC); ++j) {
                const int g = b.g_lo + (GS ? gl : (c0 - b.c_lo + j) / p.Cg);
                st.m[j] = p.mean[n * p.G + g];
                st.r[j] = p.rstd[n * p.G + g];
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) { a[j] = p.gamma[c0 + j] * st.rstd(j); be[j] = p.beta[c0 + j]; sa[j] = sb[j] = 0.f; }
            act_choice<ACT>(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    float x[VEC], z[VEC], g[VEC];
                    if (!(active && pos + i * p.P <= last)) d[i].v = typename VecOf<T, VEC>::raw{};
                    xv[i].get(x);
                    d[i].get(g);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) { x[j] -= st.mean(j); z[j] = fmaf(x[j], a[j], be[j]); }
                    act_grad_mul<T, decltype(act)::value>(g, z);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        sa[j] += g[j]; sb[j] = fmaf(g[j], x[j], sb[j]);
                        dz[i][j] = g[j];
                    }
                    xv[i].keep();
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
#pragma unroll
            for (int j = 0; j < VEC; ++j) sb[j] *= st.rstd(j);
            gn_columns<VEC>(p, sa, sb, red, tot, lv, r);
        }
        for (int k = threadIdx.x; k < cols; k += GTB) {
            float2 t = acc[k];
            for (int u = 0; u < p.NSUB; ++u) { t.x += tot[u * cols + k].x; t.y += tot[u * cols + k].y; }
            acc[k] = t;
        }
        const int pairs = p.NSUB * b.ng;
        const int L = pair_lanes<GTB>(pairs, b.cw), l = (int)threadIdx.x & (L - 1);
        for (int k = (int)threadIdx.x / L; k < pairs; k += GTB / L) {
            const int u = k / b.ng, g = k - u * b.ng;
            float2 s = make_float2(0.f, 0.f);
            for (int c = g * b.cw + l; c < (g + 1) * b.cw; c += L) {
                const float2 t = tot[u * cols + c];
                const float w = p.gamma[b.c_lo + c];
                s.x = fmaf(w, t.x, s.x); s.y = fmaf(w, t.y, s.y);
            }
            for (int o = L >> 1; o > 0; o >>= 1) { s.x += __shfl_xor(s.x, o, 64); s.y += __shfl_xor(s.y, o, 64); }
            if (l == 0) grp[k] = s;
        }
        __syncthreads();
        asm volatile("" : "+v"(pos));
        GnStat<VEC, GS> cc;                      // c1, c2 of the groups
#pragma unroll
        for (int j = 0; j < (GS ? 1 : VEC); ++j) {
            const float2 t = grp[min(sub, p.NSUB - 1) * b.ng + (GS ? gl : (c0 - b.c_lo + j) / p.Cg)];
            cc.m[j] = st.r[j] * t.x * inv_m;
            cc.r[j] = st.r[j] * st.r[j] * (t.y * inv_m);
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int s = pos + i * p.P;
            float x[VEC], g[VEC];
            xv[i].get(x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[j] = fmaf(st.mean(j) - x[j], cc.rstd(j), fmaf(a[j], dz[i][j], -cc.mean(j)));
            typename VecOf<T, VEC>::raw o;
            vec_put(o, g);
            if (active && s <= last) *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();                              // red, tot and grp are free again
    }
    for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += GTB) p.part[first * p.C + b.c_lo + k] = acc[k];
}

// f(x, dy, s) for positions s, s + P, ... below s_hi, U of them loaded at a time
template <class T, int VEC, bool CK, class F> __device__ __forceinline__ void gn_walk(const GnP& p, long long n, int s, int s_hi, int c0, F&& f) {
    for (; s < s_hi; s += U * p.P) {
        typename std::conditional<CK, CkData<VEC>, GnData<T, VEC>>::type xv[U];
        GnData<T, VEC> d[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = s + u * p.P;
            if (t < s_hi) {
                if constexpr (CK) xv[u].load(p.q, p.e, n * p.S + t, p.C, p.nb, c0);
                else xv[u].load(p.x, n * p.xn + t * p.xs + c0);
                d[u].load(p.dy, n * p.dn + t * p.ds + c0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = s + u * p.P;
            if (t < s_hi) {
                float x[VEC], g[VEC];
                xv[u].get(x);
                d[u].get(g);
                f(x, g, t);
            }
        }
    }
}

// Chunked form, first launch: column sums of a chunk of positions in part[(n nchunk + chunk) C + c].
template <class T, int VEC, bool GS, bool CK> __global__ __launch_bounds__(GTB) void gn_bwd_sums_kernel(const GnP p) {
    extern __shared__ float lds[];
    const int cols = p.LV * VEC;
    float2* red = (float2*)lds;
    float2* tot = red + (p.shuf ? GTB / 64 : p.P) * cols;
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const int chunk = (int)(t_ % p.nchunk);
    const long long n = t_ / p.nchunk;
    const GnBlock b = gn_block(p, cb);
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int c0 = b.c_lo + lv * VEC;
    float sa[VEC], sb[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) sa[j] = sb[j] = 0.f;
    if (r < p.P && c0 < b.c_hi) {
        GnStat<VEC, GS> st;
        float a[VEC], be[VEC];
#pragma unroll
        for (int j = 0; j < (GS ? 1 : VEC); ++j) {
            const int g = b.g_lo + (p.pieces == 1 ? (lv * VEC + j) / p.Cg : 0);
            st.m[j] = p.mean[n * p.G + g];
            st.r[j] = p.rstd[n * p.G + g];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) { a[j] = p.gamma[c0 + j] * st.rstd(j); be[j] = p.beta[c0 + j]; }
        const int s_hi = min(p.S, (chunk + 1) * p.chunk);
        with_act(p.act, [&](auto act) __attribute__((always_inline)) {
            gn_walk<T, VEC, CK>(p, n, chunk * p.chunk + r, s_hi, c0, [&](float (&x)[VEC], float (&g)[VEC], int s) __attribute__((always_inline)) {
                float z[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) { x[j] -= st.mean(j); z[j] = fmaf(x[j], a[j], be[j]); }
                act_grad_mul<T, decltype(act)::value>(g, z);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { sa[j] += g[j]; sb[j] = fmaf(g[j], x[j], sb[j]); }
            });
        });
#pragma unroll
        for (int j = 0; j < VEC; ++j) sb[j] *= st.rstd(j);
    }
    gn_columns<VEC>(p, sa, sb, red, tot, lv, r);
    for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += GTB) p.part[(n * p.nchunk + chunk) * p.C + b.c_lo + k] = tot[k];
}

// Chunked form, second launch: s1 and s2 of this block's groups from the column sums of every chunk, then dx.
template <class T, int VEC, bool GS, bool CK> __global__ __launch_bounds__(GTB) void gn_bwd_apply_kernel(const GnP p) {
    extern __shared__ float lds[];
    float2* grp = (float2*)lds;
    const long long lb = xcd_order(blockIdx.x, p.blocks);
    const int cb = (int)(lb % p.ncb);
    const long long t_ = lb / p.ncb;
    const int chunk = (int)(t_ % p.nchunk);
    const long long n = t_ / p.nchunk;
    const GnBlock b = gn_block(p, cb);
    const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
    for (int g = threadIdx.x >> 6; g < b.ng; g += GTB / 64) {
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
    GnStat<VEC, GS> st, cc;
#pragma unroll
    for (int j = 0; j < (GS ? 1 : VEC); ++j) {
        const int g = p.pieces == 1 ? (lv * VEC + j) / p.Cg : 0;
        st.m[j] = p.mean[n * p.G + b.g_lo + g];
        st.r[j] = p.rstd[n * p.G + b.g_lo + g];
        cc.m[j] = st.r[j] * grp[g].x; cc.r[j] = st.r[j] * st.r[j] * grp[g].y;
    }
    float a[VEC], be[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { a[j] = p.gamma[c0 + j] * st.rstd(j); be[j] = p.beta[c0 + j]; }
    const int s_hi = min(p.S, (chunk + 1) * p.chunk);
    with_act(p.act, [&](auto act) __attribute__((always_inline)) {
        gn_walk<T, VEC, CK>(p, n, chunk * p.chunk + r, s_hi, c0, [&](float (&x)[VEC], float (&g)[VEC], int s) __attribute__((always_inline)) {
            float z[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) { x[j] -= st.mean(j); z[j] = fmaf(x[j], a[j], be[j]); }
            act_grad_mul<T, decltype(act)::value>(g, z);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[j] = fmaf(-x[j], cc.rstd(j), fmaf(a[j], g[j], -cc.mean(j)));
            typename VecOf<T, VEC>::raw o;
            vec_put(o, g);
            *(typename VecOf<T, VEC>::raw*)((T*)p.y + n * p.yn + s * p.ys + c0) = o;
        });
    });
}

template <class T, int VEC, bool GS, bool CK> int gn_bwd_t(const GnP& p, const GnPlan& pl, hipStream_t st) {
    const int cols = p.LV * VEC;
    const size_t lds = sizeof(float2) * ((size_t)(p.shuf ? GTB / 64 : p.P * p.NSUB) * cols + 2 * (size_t)p.NSUB * cols + cols);
    if (!pl.held) {
        const int rc = gn_launch(gn_bwd_sums_kernel<T, VEC, GS, CK>, p, GTB, lds, st);
        if (rc != FAVAE_OK) return rc;
        return gn_launch(gn_bwd_apply_kernel<T, VEC, GS, CK>, p, GTB, sizeof(float2) * cdiv(p.CB, std::min(p.Cg, p.CB)), st);
    }
    if constexpr (VEC * sizeof(T) == 16) {
        int rc = FAVAE_OK;
        with_act_host(p.act, [&](auto act) {
            constexpr int A = decltype(act)::value;
            if (pl.items <= 4) rc = gn_launch(gn_bwd_kernel<T, VEC, 4, GS, CK, A>, p, GTB, lds, st);
            else if (pl.items <= 8) rc = gn_launch(gn_bwd_kernel<T, VEC, 8, GS, CK, A>, p, GTB, lds, st);
            else rc = gn_launch(gn_bwd_kernel<T, VEC, ITEMS_MAX, GS, CK, A>, p, GTB, lds, st);
        });
        return rc;
    } else {
        return pl.items <= 4 ? gn_launch(gn_bwd_kernel<T, VEC, 4, GS, CK, -1>, p, GTB, lds, st)
                             : gn_launch(gn_bwd_kernel<T, VEC, ITEMS_MAX, GS, CK, -1>, p, GTB, lds, st);
    }
}
template <class T, bool CK> int gn_bwd(const GnP& p, const GnPlan& pl, hipStream_t st) {
#define GN_F(T_, V) { if constexpr (V == 1) return gn_bwd_t<T_, V, true, CK>(p, pl, st); else return pl.gs ? gn_bwd_t<T_, V, true, CK>(p, pl, st) : gn_bwd_t<T_, V, false, CK>(p, pl, st); }
    GN_VEC(T, pl.vec, GN_F);
#undef GN_F
}

}  // namespace
