// Backward kernels of group norm with an activation (formulas and the four forms: groupnorm.hip).
#pragma once
#include "groupnorm.h"

namespace {

template <class T, bool TAIL, bool CK> using GnX = typename std::conditional<CK, CkData<T, TAIL>, GnData<T, TAIL>>::type;
template <class T, bool TAIL, bool CK>
__device__ __forceinline__ void gn_load(const GnP& p, GnX<T, TAIL, CK>& x, GnData<T, TAIL>& d, long long n, int s, const GnLane<T, TAIL>& l) {
    if constexpr (CK) x.load(p.q, p.e, n * p.S + s, p.C, p.nb, l);
    else x.load(p.x, n * p.xn + s * p.xs + l.c0, l);
    d.load(p.dy, n * p.dn + s * p.ds + l.c0, l);
}

// ---- wave form -----------------------------------------------------------------------------------------------------------
// (lanes as in gn_wave_fwd_kernel.)  dz is held: its exp and reciprocal are half the work of a pass.  The sums over samples stay in each lane's
// registers to the end; the waves of a workgroup then leave one row of them, part[row C + c].
template <class T, int ITEMS, int GPV, bool CK> __global__ __launch_bounds__(256) void gn_wave_bwd_kernel(const GnP p) {
    constexpr int VEC = VEC16<T>;
    __shared__ float2 red[4][64][VEC + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const unsigned lb = xcd_order(blockIdx.x, (unsigned)p.blocks), row_ = lb / (unsigned)p.ncb;
    const int cb = (int)(lb - row_ * p.ncb);
    const long long row = row_, rows = (unsigned)p.blocks / (unsigned)p.ncb;
    const int lv = lane & (p.LV - 1), pos = lane / p.LV, gl = GPV == 1 ? p.Cg / VEC : 1;
    const bool col_ok = cb * p.CB + lv * VEC < p.C;
    const GnLane<T, false> ln(min(cb * p.CB + lv * VEC, p.C - VEC), p.C, 0);
    const int c0 = ln.c0, g0 = c0 / p.Cg;
    const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
    float ga[VEC], be[VEC], sa[VEC], sb[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { ga[j] = p.gamma[c0 + j]; be[j] = p.beta[c0 + j]; sa[j] = sb[j] = 0.f; }
    with_act(p.act, [&](auto act) __attribute__((always_inline)) {
        for (long long n = row * waves + wave; n < p.N; n += rows * waves) {
            GnX<T, false, CK> xv[ITEMS];
            GnData<T, false> d[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) gn_load<T, false, CK>(p, xv[i], d[i], n, min(pos + i * p.P, p.S - 1), ln);
            GnStat<VEC, GPV> st;
#pragma unroll
            for (int j = 0; j < GPV; ++j) { st.m[j] = p.mean[n * p.G + g0 + j]; st.r[j] = p.rstd[n * p.G + g0 + j]; }
            float dz[ITEMS][VEC], la[VEC], lb_[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) la[j] = lb_[j] = 0.f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                float x[VEC], z[VEC];
                if (pos + i * p.P >= p.S) d[i].v = make_uint4(0u, 0u, 0u, 0u);       // a position that is not there counts for nothing
                xv[i].get(x);
                d[i].get(dz[i]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { x[j] -= st.mean(j); z[j] = fmaf(x[j], ga[j] * st.rstd(j), be[j]); }
                act_grad_mul<T, decltype(act)::value>(dz[i], z);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { la[j] += dz[i][j]; lb_[j] = fmaf(dz[i][j], x[j], lb_[j]); }
                xv[i].keep();
                __builtin_amdgcn_sched_barrier(0);       // one item after the other: interleaved they need the registers of all
            }
            float s1[GPV], s2[GPV];
#pragma unroll
            for (int j = 0; j < GPV; ++j) s1[j] = s2[j] = 0.f;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                lb_[j] *= st.rstd(j);
                sa[j] += la[j]; sb[j] += lb_[j];
                s1[j * GPV / VEC] = fmaf(ga[j], la[j], s1[j * GPV / VEC]);
                s2[j * GPV / VEC] = fmaf(ga[j], lb_[j], s2[j * GPV / VEC]);
            }
#pragma unroll
            for (int j = 0; j < GPV; ++j) {
                for (int o = p.LV; o < 64; o <<= 1) { s1[j] += __shfl_xor(s1[j], o, 64); s2[j] += __shfl_xor(s2[j], o, 64); }
                if constexpr (GPV == 1)
                    for (int o = 1; o < gl; o <<= 1) { s1[j] += __shfl_xor(s1[j], o, 64); s2[j] += __shfl_xor(s2[j], o, 64); }
                s1[j] *= st.r[j] * inv_m;                                            // c1, c2
                s2[j] *= st.r[j] * st.r[j] * inv_m;
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int s = pos + i * p.P;
                float x[VEC], g[VEC];
                xv[i].get(x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) g[j] = fmaf(st.mean(j) - x[j], s2[j * GPV / VEC], fmaf(ga[j] * st.rstd(j), dz[i][j], -s1[j * GPV / VEC]));
                uint4 o;
                vec_put(o, g);
                if (col_ok && s < p.S) ln.store(p.y, n * p.yn + s * p.ys + c0, o);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    });
    for (int o = p.LV; o < 64; o <<= 1)
#pragma unroll
        for (int j = 0; j < VEC; ++j) { sa[j] += __shfl_xor(sa[j], o, 64); sb[j] += __shfl_xor(sb[j], o, 64); }
    if (pos == 0)
#pragma unroll
        for (int j = 0; j < VEC; ++j) red[wave][lv][j] = make_float2(sa[j], sb[j]);
    lds_barrier();
    if (wave == 0 && pos == 0 && col_ok)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float2 t = red[0][lv][j];
            for (int w = 1; w < waves; ++w) { t.x += red[w][lv][j].x; t.y += red[w][lv][j].y; }
            p.part[row * p.C + c0 + j] = t;
        }
}

// ---- piped form ----------------------------------------------------------------------------------------------------------
// The block takes channel block blockIdx % ncb of samples blockIdx / ncb, + gridDim / ncb, ...  dy, and x unless it is a checkpoint, come through
// LDS, where a wave reads back what its own DMA brought, so that only the sums need barriers; a checkpoint's 9 bytes a vector and the statistics
// of the next sample wait in registers.  Stores go through a descriptor too, lanes without a position storing nowhere: the loads of the next
// sample are then older than exactly ITEMS stores, and the wait at a sample's end, for all but ITEMS operations, holds for the loads whatever became
// of the stores.  Column sums over the block's samples go to part[row C + c].
// What overlaps is the next sample's loads and the first pass over the present one (dz and its column sums): the staging buffers and the sums are one
// LDS array, so the compiler takes every access to red, tot and grp for one that the DMA may meet, and waits for all vector memory before the first
// of them and at the top of the loop.  512 x 1024 x 128 bf16 95 us (156 held), 256 x 1024 x 128 45, from a checkpoint as well, 3.8 TB/s.
// <bf16, 8 groups a vector, checkpoint> spills 20 to 25 registers with an activation.
template <class T, int GPV, bool CK, int ACT> __global__ __launch_bounds__(GTP) void gn_piped_bwd_kernel(const GnP p) {
    extern __shared__ float lds[];
    constexpr int VEC = VEC16<T>, ITEMS = PIPED_ITEMS;
    constexpr long long ES = sizeof(T);
    const int cols = p.LV * VEC;
    char* dbuf = (char*)lds;
    char* xbuf = dbuf + ITEMS * GTP * 16;
    float2* red = (float2*)(xbuf + (CK ? 0 : ITEMS * GTP * 16));      // [GTP / 64][cols]
    float2* tot = red + (GTP / 64) * cols;                            // [cols]
    float2* grp = tot + cols;                                         // [ng]
    float2* acc = grp + cols;                                         // [cols]
    float* gam = (float*)(acc + cols);                                // [cols]
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const unsigned lb = xcd_order(blockIdx.x, (unsigned)p.blocks), row_ = lb / (unsigned)p.ncb;
    const int cb = (int)(lb - row_ * p.ncb);
    const long long row = row_, stride = (unsigned)p.blocks / (unsigned)p.ncb;
    const GnBlock b = gn_block(p, cb);
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const bool has = b.c_lo + lv * VEC < b.c_hi;
    const GnLane<T, false> ln(min(b.c_lo + lv * VEC, b.c_hi - VEC), b.c_hi, 0);
    const int c0 = ln.c0, mine = has ? (p.S - r + p.P - 1) / p.P : 0;
    const unsigned dof = (unsigned)((r * p.ds + c0) * ES), dstep = (unsigned)(p.P * p.ds * ES);
    const unsigned xof = (unsigned)((r * p.xs + c0) * ES), xstep = (unsigned)(p.P * p.xs * ES);
    const unsigned yof = (unsigned)((r * p.ys + c0) * ES), ystep = (unsigned)(p.P * p.ys * ES);
    int gi[GPV];
    group_of<VEC / GPV>(gi, c0 - b.c_lo, p.Cg, b.ng - 1);
    float ga[VEC], be[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { ga[j] = p.gamma[c0 + j]; be[j] = p.beta[c0 + j]; }
    for (int k = threadIdx.x; k < cols; k += GTP) {
        acc[k] = make_float2(0.f, 0.f);
        gam[k] = b.c_lo + k < b.c_hi ? p.gamma[b.c_lo + k] : 0.f;
    }
    const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
    GnStat<VEC, GPV> nst;
    CkData<T, false> nx[CK ? ITEMS : 1];
    const auto fetch = [&](long long n) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < GPV; ++j) { nst.m[j] = p.mean[n * p.G + b.g_lo + gi[j]]; nst.r[j] = p.rstd[n * p.G + b.g_lo + gi[j]]; }
        if constexpr (CK) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) nx[i].load(p.q, p.e, n * p.S + min(r + i * p.P, p.S - 1), p.C, p.nb, ln);
        } else gn_dma<ITEMS>(xbuf, wave, gn_rsrc(p.x, n * p.xn * ES), xof, xstep, mine);
        gn_dma<ITEMS>(dbuf, wave, gn_rsrc(p.dy, n * p.dn * ES), dof, dstep, mine);
    };
    long long n = row;
    fetch(n);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    for (; n < p.N; n += stride) {
        GnData<T, false> d[ITEMS];
        GnX<T, false, CK> xv[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            d[i].v = *(const uint4*)(dbuf + (i * GTP + (int)threadIdx.x) * 16);
            if constexpr (CK) xv[i] = nx[i];
            else xv[i].v = *(const uint4*)(xbuf + (i * GTP + (int)threadIdx.x) * 16);
        }
        const GnStat<VEC, GPV> st = nst;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");            // the buffers are read: the next sample may come
        if (n + stride < p.N) fetch(n + stride);
        float a[VEC], dz[ITEMS][VEC];
        {
            float sa[VEC], sb[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) { a[j] = ga[j] * st.rstd(j); sa[j] = sb[j] = 0.f; }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                float x[VEC], z[VEC], g[VEC];
                xv[i].get(x);
                d[i].get(g);                                          // (zeros where there is no position)
#pragma unroll
                for (int j = 0; j < VEC; ++j) { x[j] -= st.mean(j); z[j] = fmaf(x[j], a[j], be[j]); }
                act_grad_mul<T, ACT>(g, z);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    sa[j] += g[j]; sb[j] = fmaf(g[j], x[j], sb[j]);
                    dz[i][j] = g[j];
                }
                xv[i].keep();
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) sb[j] *= st.rstd(j);
            // sums of the rows of a wave by shuffles, of the waves in LDS
            for (int o = p.LV; o < 64; o <<= 1)
#pragma unroll
                for (int j = 0; j < VEC; ++j) { sa[j] += __shfl_xor(sa[j], o, 64); sb[j] += __shfl_xor(sb[j], o, 64); }
            if ((int)(threadIdx.x & 63) < p.LV && has)
#pragma unroll
                for (int j = 0; j < VEC; ++j) red[wave * cols + lv * VEC + j] = make_float2(sa[j], sb[j]);
        }
        lds_barrier();
        for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += GTP) {
            float2 s = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < GTP / 64; ++w) { const float2 t = red[w * cols + k]; s.x += t.x; s.y += t.y; }
            const float2 u = acc[k];
            acc[k] = make_float2(u.x + s.x, u.y + s.y);
            tot[k] = make_float2(gam[k] * s.x, gam[k] * s.y);
        }
        lds_barrier();
        const int ls = pair_lanes_log2(GTP, b.ng, b.cw), L = 1 << ls, l = (int)threadIdx.x & (L - 1);
        for (int g = (int)threadIdx.x >> ls; g < b.ng; g += GTP >> ls) {
            float2 s = make_float2(0.f, 0.f);
            for (int c = g * b.cw + l; c < (g + 1) * b.cw; c += L) { s.x += tot[c].x; s.y += tot[c].y; }
            for (int o = L >> 1; o > 0; o >>= 1) { s.x += __shfl_xor(s.x, o, 64); s.y += __shfl_xor(s.y, o, 64); }
            if (l == 0) grp[g] = s;
        }
        lds_barrier();
        GnStat<VEC, GPV> cc;                                          // c1, c2 of the groups
#pragma unroll
        for (int j = 0; j < GPV; ++j) {
            const float2 t = grp[gi[j]];
            cc.m[j] = st.r[j] * t.x * inv_m;
            cc.r[j] = st.r[j] * st.r[j] * (t.y * inv_m);
        }
        const __amdgpu_buffer_rsrc_t ry = gn_rsrc(p.y, n * p.yn * ES);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            float x[VEC], g[VEC];
            xv[i].get(x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[j] = fmaf(st.mean(j) - x[j], cc.rstd(j), fmaf(a[j], dz[i][j], -cc.mean(j)));
            uint4 o;
            vec_put(o, g);
            __builtin_amdgcn_raw_buffer_store_b128(gn_v4u{o.x, o.y, o.z, o.w}, ry, (int)(i < mine ? yof + i * ystep : GN_NOWHERE), 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ITEMS) : "memory");
    }
    lds_barrier();
    for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += GTP) p.part[row * p.C + b.c_lo + k] = acc[k];
}

// ---- workgroup forms -----------------------------------------------------------------------------------------------------
// Column sums (dz, dz xh) of a block's threads into tot[sub][CB] (float2).  red: [rows][CB] float2.
template <int VEC, class O>
__device__ __forceinline__ void gn_columns(const GnP& p, float (&a)[VEC], float (&bq)[VEC], float2* red, float2* tot, int col, int r, O&& own) {
    const int cols = p.LV * VEC;
    int rows = p.P;
    if (p.shuf) {
        for (int o = p.LV; o < 64; o <<= 1)
#pragma unroll
            for (int j = 0; j < VEC; ++j) { a[j] += __shfl_xor(a[j], o, 64); bq[j] += __shfl_xor(bq[j], o, 64); }
        rows = p.nt / 64;
        if ((int)(threadIdx.x & 63) < p.LV)
#pragma unroll
            for (int j = 0; j < VEC; ++j) if (own(j)) red[(threadIdx.x >> 6) * cols + col + j] = make_float2(a[j], bq[j]);
    } else if (r < p.P * p.NSUB) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) if (own(j)) red[r * cols + col + j] = make_float2(a[j], bq[j]);
    }
    lds_barrier();
    for (int k = threadIdx.x; k < p.NSUB * cols; k += p.nt) {
        const int sub = k / cols, c = k - sub * cols;
        float2 s = make_float2(0.f, 0.f);
        for (int i = 0; i < rows; ++i) {
            const float2 t = red[(sub * rows + i) * cols + c];
            s.x += t.x; s.y += t.y;
        }
        tot[k] = s;
    }
    lds_barrier();
}
// gamma rstd and beta of a thread's channels
template <int VEC, int GPV, bool TAIL>
__device__ __forceinline__ void gn_affine(const GnP& p, const GnStat<VEC, GPV>& st, int c0, float (&a)[VEC], float (&be)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int c = TAIL ? min(c0 + j, p.C - 1) : c0 + j;
        a[j] = p.gamma[c] * st.rstd(j);
        be[j] = p.beta[c];
    }
}

// Held form: the block takes samples blockIdx, + gridDim, ...: dx, and its column sums over all of them in part[blockIdx C + c].
// ACT: the activation (chosen inside the kernel it would cost the last registers).
// Lanes without a channel, a sample or a position read the last valid one instead and count for nothing, so that only stores are
// under a lane mask.  Items are kept one after the other: interleaved by the compiler they would need the registers of all at once.
template <class T, int ITEMS, int GPV, bool TAIL, bool CK, int ACT> __global__ __launch_bounds__(GTB) void gn_bwd_kernel(const GnP p) {
    extern __shared__ float lds[];
    constexpr int VEC = VEC16<T>;
    const int cols = p.LV * VEC;
    float2* red = (float2*)lds;
    float2* tot = red + (p.shuf ? (p.nt / 64) * cols : p.P * p.NSUB * cols);
    float2* grp = tot + p.NSUB * cols;           // [NSUB][ng]
    float2* acc = grp + p.NSUB * cols;           // [cols]
    const unsigned lb = xcd_order(blockIdx.x, (unsigned)p.blocks), row_ = lb / (unsigned)p.ncb;
    const int cb = (int)(lb - row_ * p.ncb);
    const long long first = row_, stride = (unsigned)p.blocks / (unsigned)p.ncb;
    const GnBlock b = gn_block(p, cb);
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int sub = r / p.P;
    int pos = r - sub * p.P;
    const int last = p.S - 1;
    const bool has = b.c_lo + lv * VEC < b.c_hi, col_ok = sub < p.NSUB && has;
    const GnLane<T, TAIL> ln(b.c_lo, b.c_hi, min(lv, (b.c_hi - b.c_lo - 1) / VEC));
    const int c0 = ln.c0;
    const auto own = [&](int j) { return has && ln.own(j); };
    int gi[GPV];
    group_of<1>(gi, c0 - b.c_lo, p.Cg, b.ng - 1);
    for (int k = threadIdx.x; k < cols; k += p.nt) acc[k] = make_float2(0.f, 0.f);
    const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
    for (long long nb0 = first; nb0 * p.NSUB < p.N; nb0 += stride) {
        const long long n0 = nb0 * p.NSUB + sub, n = min(n0, (long long)p.N - 1);
        const bool active = col_ok && n0 < p.N;
        asm volatile("" : "+v"(pos));            // the items' offsets are made where they are used, not kept over the samples
        GnData<T, TAIL> d[ITEMS];
        GnX<T, TAIL, CK> xv[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) gn_load<T, TAIL, CK>(p, xv[i], d[i], n, min(pos + i * p.P, last), ln);
        GnStat<VEC, GPV> st;
        float a[VEC];                            // gamma rstd
        float dz[ITEMS][VEC];                    // held: its exp and reciprocal are half the work of a pass
        {
            float be[VEC], sa[VEC], sb[VEC];
#pragma unroll
            for (int j = 0; j < GPV; ++j) { st.m[j] = p.mean[n * p.G + b.g_lo + gi[j]]; st.r[j] = p.rstd[n * p.G + b.g_lo + gi[j]]; }
            gn_affine<VEC, GPV, TAIL>(p, st, c0, a, be);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sa[j] = sb[j] = 0.f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                float x[VEC], z[VEC], g[VEC];
                if (!(active && pos + i * p.P <= last)) d[i].v = make_uint4(0u, 0u, 0u, 0u);
                xv[i].get(x);
                d[i].get(g);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { x[j] -= st.mean(j); z[j] = fmaf(x[j], a[j], be[j]); }
                act_grad_mul<T, ACT>(g, z);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    sa[j] += g[j]; sb[j] = fmaf(g[j], x[j], sb[j]);
                    dz[i][j] = g[j];
                }
                xv[i].keep();
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) sb[j] *= st.rstd(j);
            gn_columns<VEC>(p, sa, sb, red, tot, c0 - b.c_lo, r, own);
        }
        for (int k = threadIdx.x; k < cols; k += p.nt) {
            float2 t = acc[k];
            for (int u = 0; u < p.NSUB; ++u) { t.x += tot[u * cols + k].x; t.y += tot[u * cols + k].y; }
            acc[k] = t;
        }
        const int pairs = p.NSUB * b.ng;
        const int ls = pair_lanes_log2(p.nt, pairs, b.cw), L = 1 << ls, l = (int)threadIdx.x & (L - 1);
        for (int k = (int)threadIdx.x >> ls; k < pairs; k += p.nt >> ls) {
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
        lds_barrier();
        asm volatile("" : "+v"(pos));
        GnStat<VEC, GPV> cc;                     // c1, c2 of the groups
#pragma unroll
        for (int j = 0; j < GPV; ++j) {
            const float2 t = grp[min(sub, p.NSUB - 1) * b.ng + gi[j]];
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
            uint4 o;
            vec_put(o, g);
            if (active && s <= last) ln.store_whole(p.y, n * p.yn + s * p.ys + c0, o);
            __builtin_amdgcn_sched_barrier(0);
        }
        lds_barrier();                           // red, tot and grp are free again
    }
    for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += p.nt) p.part[first * p.C + b.c_lo + k] = acc[k];
}

// f(x, dy, s) for positions s, s + P, ... below s_hi, GU of them loaded at a time
template <class T, bool TAIL, bool CK, class F> __device__ __forceinline__ void gn_walk(const GnP& p, long long n, int s, int s_hi, const GnLane<T, TAIL>& l, F&& f) {
    for (; s < s_hi; s += GU * p.P) {
        GnX<T, TAIL, CK> xv[GU];
        GnData<T, TAIL> d[GU];
#pragma unroll
        for (int u = 0; u < GU; ++u)
            if (s + u * p.P < s_hi) gn_load<T, TAIL, CK>(p, xv[u], d[u], n, s + u * p.P, l);
#pragma unroll
        for (int u = 0; u < GU; ++u) {
            const int t = s + u * p.P;
            if (t < s_hi) {
                float x[VEC16<T>], g[VEC16<T>];
                xv[u].get(x);
                d[u].get(g);
                f(x, g, t);
            }
        }
    }
}

// The first launch goes over the chunks from the back: what was written last, and for the launch that comes after it what was read last, is still in
// the 256 MB cache (512 x 4096 x 64 bf16 in a loop: 110 and 139 us, 127 and 150 with both from the front).
struct GnChunk { int cb, chunk; long long n; };
__device__ __forceinline__ GnChunk gn_chunk(const GnP& p, bool back) {
    const unsigned lb = xcd_order(back ? (unsigned)p.blocks - 1u - blockIdx.x : blockIdx.x, (unsigned)p.blocks), t = lb / (unsigned)p.ncb, n = t / (unsigned)p.nchunk;
    return {(int)(lb - t * p.ncb), (int)(t - n * p.nchunk), (long long)n};
}

// Chunked form, first launch: column sums of a chunk of positions in part[(n nchunk + chunk) C + c].
template <class T, int GPV, bool TAIL, bool CK> __global__ __launch_bounds__(GTB) void gn_bwd_sums_kernel(const GnP p) {
    extern __shared__ float lds[];
    constexpr int VEC = VEC16<T>;
    const int cols = p.LV * VEC;
    float2* red = (float2*)lds;
    float2* tot = red + (p.shuf ? p.nt / 64 : p.P) * cols;
    const GnChunk k_ = gn_chunk(p, true);
    const GnBlock b = gn_block(p, k_.cb);
    const long long n = k_.n;
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const bool has = b.c_lo + lv * VEC < b.c_hi;
    const GnLane<T, TAIL> ln(b.c_lo, b.c_hi, lv);
    const int c0 = ln.c0;
    const auto own = [&](int j) { return has && ln.own(j); };
    float sa[VEC], sb[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) sa[j] = sb[j] = 0.f;
    if (r < p.P && has) {
        GnStat<VEC, GPV> st;
        float a[VEC], be[VEC];
        int gi[GPV];
        group_of<1>(gi, p.pieces == 1 ? c0 - b.c_lo : 0, p.Cg, b.ng - 1);
#pragma unroll
        for (int j = 0; j < GPV; ++j) {
            const int g = b.g_lo + gi[j];
            st.m[j] = p.mean[n * p.G + g];
            st.r[j] = p.rstd[n * p.G + g];
        }
        gn_affine<VEC, GPV, TAIL>(p, st, c0, a, be);
        with_act(p.act, [&](auto act) __attribute__((always_inline)) {
            gn_walk<T, TAIL, CK>(p, n, k_.chunk * p.chunk + r, min(p.S, (k_.chunk + 1) * p.chunk), ln, [&](float (&x)[VEC], float (&g)[VEC], int s) __attribute__((always_inline)) {
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
    gn_columns<VEC>(p, sa, sb, red, tot, c0 - b.c_lo, r, own);
    for (int k = threadIdx.x; k < b.c_hi - b.c_lo; k += p.nt) p.part[(n * p.nchunk + k_.chunk) * p.C + b.c_lo + k] = tot[k];
}

// Chunked form, third launch: dx.
template <class T, int GPV, bool TAIL, bool CK> __global__ __launch_bounds__(GTB) void gn_bwd_apply_kernel(const GnP p) {
    constexpr int VEC = VEC16<T>;
    const GnChunk k_ = gn_chunk(p, false);
    const GnBlock b = gn_block(p, k_.cb);
    const long long n = k_.n;
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    if (r >= p.P || b.c_lo + lv * VEC >= b.c_hi) return;
    const GnLane<T, TAIL> ln(b.c_lo, b.c_hi, lv);
    const int c0 = ln.c0;
    GnStat<VEC, GPV> st, cc;
    int gi[GPV];
    group_of<1>(gi, p.pieces == 1 ? c0 - b.c_lo : 0, p.Cg, b.ng - 1);
#pragma unroll
    for (int j = 0; j < GPV; ++j) {
        const long long g = n * p.G + b.g_lo + gi[j];
        st.m[j] = p.mean[g];
        st.r[j] = p.rstd[g];
        const float2 t = p.s12[g];
        cc.m[j] = st.r[j] * t.x;
        cc.r[j] = st.r[j] * st.r[j] * t.y;
    }
    float a[VEC], be[VEC];
    gn_affine<VEC, GPV, TAIL>(p, st, c0, a, be);
    with_act(p.act, [&](auto act) __attribute__((always_inline)) {
        gn_walk<T, TAIL, CK>(p, n, k_.chunk * p.chunk + r, min(p.S, (k_.chunk + 1) * p.chunk), ln, [&](float (&x)[VEC], float (&g)[VEC], int s) __attribute__((always_inline)) {
            float z[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) { x[j] -= st.mean(j); z[j] = fmaf(x[j], a[j], be[j]); }
            act_grad_mul<T, decltype(act)::value>(g, z);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[j] = fmaf(-x[j], cc.rstd(j), fmaf(a[j], g[j], -cc.mean(j)));
            uint4 o;
            vec_put(o, g);
            ln.store(p.y, n * p.yn + s * p.ys + c0, o);
        });
    });
}

// Sums over the rows of part [rows][C].  Blocks below gblocks (chunked form, second launch): (s1, s2) / m of a group a wave, from the
// sample's nchunk rows.  The others: dbeta, dgamma of 4 channels, 256 rows at a time.
__global__ __launch_bounds__(1024) void gn_join_kernel(const GnP p, long long rows, int gblocks, float* dgamma, float* dbeta) {
    __shared__ float2 red[16][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x < gblocks) {
        const long long g = (long long)blockIdx.x * 16 + wave;
        if (g >= (long long)p.N * p.G) return;
        const long long n = (unsigned)g / (unsigned)p.G;
        const int c0 = (int)(g - n * p.G) * p.Cg, dch = 64 / p.Cg, dc = 64 - dch * p.Cg;
        int ch = lane / p.Cg, c1 = lane - ch * p.Cg;
        float2 s = make_float2(0.f, 0.f);
        while (ch < p.nchunk) {
            const int c = c0 + c1;
            const float2 t = p.part[(n * p.nchunk + ch) * p.C + c];
            const float w = p.gamma[c];
            s.x = fmaf(w, t.x, s.x); s.y = fmaf(w, t.y, s.y);
            ch += dch; c1 += dc;
            if (c1 >= p.Cg) { c1 -= p.Cg; ++ch; }
        }
        s.x = wave_total(s.x); s.y = wave_total(s.y);
        const float inv_m = 1.f / ((float)p.S * (float)p.Cg);
        if (lane == 0) p.s12[g] = make_float2(s.x * inv_m, s.y * inv_m);
        return;
    }
    const int c = ((int)blockIdx.x - gblocks) * 4 + (threadIdx.x & 3);
    float2 s = make_float2(0.f, 0.f);
    if (c < p.C)
#pragma unroll 4
        for (long long i = threadIdx.x >> 2; i < rows; i += 256) {
            const float2 t = p.part[i * p.C + c];
            s.x += t.x; s.y += t.y;
        }
#pragma unroll
    for (int o = 4; o < 64; o <<= 1) { s.x += __shfl_xor(s.x, o, 64); s.y += __shfl_xor(s.y, o, 64); }
    if (lane < 4) red[wave][lane] = s;
    lds_barrier();
    if (threadIdx.x < 4 && c < p.C) {
        float2 t = red[0][threadIdx.x];
        for (int w = 1; w < 16; ++w) { t.x += red[w][threadIdx.x].x; t.y += red[w][threadIdx.x].y; }
        if (dbeta) dbeta[c] = t.x;
        if (dgamma) dgamma[c] = t.y;
    }
}

template <class T, bool CK> int gn_bwd(const GnP& p, const GnPlan& pl, float* dgamma, float* dbeta, hipStream_t st) {
    int rc = FAVAE_OK;
    const int pblocks = dgamma || dbeta ? cdiv(p.C, 4) : 0;
    const auto join = [&](int gblocks) {
        if (gblocks + pblocks > 0) gn_join_kernel<<<gblocks + pblocks, 1024, 0, st>>>(p, pl.rows, gblocks, dgamma, dbeta);
        FAVAE_LAUNCH_CHECK();
        return FAVAE_OK;
    };
    if (pl.rows == 0) return join(0);                                    // no values: zero gradients
    if (pl.form == GN_WAVE) {
        rc = gn_wave_variants<T>(pl, [&](auto gpv, auto items) {
            return gn_launch(gn_wave_bwd_kernel<T, decltype(items)::value, decltype(gpv)::value, CK>, p, pl.threads, 0, st);
        });
        return rc != FAVAE_OK ? rc : join(0);
    }
    if (pl.form == GN_PIPED) {
        const size_t cols = (size_t)p.LV * VEC16<T>;
        const size_t lds = (size_t)(CK ? 1 : 2) * PIPED_ITEMS * GTP * 16 + sizeof(float2) * (GTP / 64 + 3) * cols + sizeof(float) * cols;
        with_act_host(p.act, [&](auto act) {
            constexpr int A = decltype(act)::value;
            rc = gn_gpv<T>(pl, [&](auto gpv) { return gn_launch(gn_piped_bwd_kernel<T, decltype(gpv)::value, CK, A>, p, GTP, lds, st); });
        });
        return rc != FAVAE_OK ? rc : join(0);
    }
    const size_t cols = (size_t)p.LV * VEC16<T>, rows = p.shuf ? p.nt / 64 : p.P * p.NSUB;
    return gn_variants<T>(pl, [&](auto gpv, auto tail) {
        constexpr int GPV = decltype(gpv)::value;
        constexpr bool TAIL = decltype(tail)::value;
        if (pl.form == GN_CHUNKED) {
            int rc = gn_launch(gn_bwd_sums_kernel<T, GPV, TAIL, CK>, p, p.nt, sizeof(float2) * (rows + 1) * cols, st);
            if (rc != FAVAE_OK) return rc;
            rc = join((int)cdivll((long long)p.N * p.G, 16));
            return rc != FAVAE_OK ? rc : gn_launch(gn_bwd_apply_kernel<T, GPV, TAIL, CK>, p, p.nt, 0, st);
        }
        const size_t lds = sizeof(float2) * (rows + 2 * p.NSUB + 1) * cols;
        int rc = FAVAE_OK;
        with_act_host(p.act, [&](auto act) {
            constexpr int A = decltype(act)::value;
            if (pl.items <= 4) rc = gn_launch(gn_bwd_kernel<T, 4, GPV, TAIL, CK, A>, p, p.nt, lds, st);
            else if (pl.items <= 8) rc = gn_launch(gn_bwd_kernel<T, 8, GPV, TAIL, CK, A>, p, p.nt, lds, st);
            else if (pl.items <= 12) rc = gn_launch(gn_bwd_kernel<T, 12, GPV, TAIL, CK, A>, p, p.nt, lds, st);
            else rc = gn_launch(gn_bwd_kernel<T, ITEMS_MAX, GPV, TAIL, CK, A>, p, p.nt, lds, st);
        });
        return rc != FAVAE_OK ? rc : join(0);
    });
}

}  // namespace
