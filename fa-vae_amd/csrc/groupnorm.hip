// Group norm with an activation over channels-last maps, forward and backward.
//
//   per sample n and group g, over the m = S * Cg values of its S positions and Cg channels:
//     mean = sum x / m,  rstd = (sum (x - mean)^2 / m + eps)^-1/2,  xh = (x - mean) rstd,  z = gamma xh + beta,  y = act(z)
//   backward:  dz = dy act'(z),  dbeta = sum dz,  dgamma = sum dz xh  (over samples and positions),
//     dx = rstd (gamma dz - (s1 + xh s2) / m),  s1 = sum over the group of gamma dz,  s2 = sum over the group of gamma dz xh
//   The kernels work with d = x - mean: z = fma(d, gamma rstd, beta), sum dz d, and dx = (gamma rstd) dz - c1 - d c2 with
//   c1 = rstd s1 / m, c2 = rstd^2 s2 / m.
//
// Memory bounds both.  Four forms:
//   wave     the positions of a run of groups fit a wave's registers (up to 8 vectors of 16 bytes a lane; small maps): every wave works for
//            itself, sums cross lanes by shuffles, there is no LDS and no barrier.
//   held     they fit a workgroup's registers (up to 16 vectors a thread): the input is read once, sums meet in LDS.
//   piped    (backward, up to 8 vectors a thread, 16-byte aligned tensors, enough samples) the same, and during the first pass over one sample
//            the next is on its way into LDS, so that memory does not idle while a CU computes: 512 x 1024 x 128 bf16 silu 156 -> 95 us.
//            (Forward two workgroups share a CU and cover each other: 68 us held, 81 piped, not kept.)
//   chunked  they do not, or there are too few groups to fill the chip: a first launch leaves the partial sums of each chunk of positions,
//            a later one joins them and makes the second pass over the data.
// The variance is the sum of squared distances from the mean (no cancellation).  Sums are fp32 within a thread and joined in a fixed
// order: the results do not depend on scheduling.
#include "groupnorm.h"
#include <numeric>

namespace {

// VEC values of a position into an 8-bit checkpoint: 32 / VEC neighbouring lanes hold a block (ck_in_kernel), all of them active
template <int VEC> __device__ __forceinline__ void ck_store(const GnP& p, float (&f)[VEC], long long pos, int c) {
    unsigned m = ck_amax(f);
#pragma unroll
    for (int o = 1; o < 32 / VEC; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    const unsigned code = ck_code(m);
    unsigned w[VEC / 4];
    ck_bytes(w, f, code);
    __builtin_memcpy(p.qo + pos * p.C + c, w, VEC);
    if ((c & 31) == 0) p.eo[pos * p.nb + (c >> 5)] = (unsigned char)code;
}

// ---- wave form -----------------------------------------------------------------------------------------------------------
// A wave takes channel block blockIdx % ncb of samples (blockIdx / ncb) * waves + wave, + rows * waves, ...  Groups of Cg = 2^k channels, or
// whole vectors of them: a group is VEC / GPV channels of a lane, or the vectors of Cg / VEC neighbouring lanes.
template <class T, int ITEMS, int GPV> __global__ __launch_bounds__(256) void gn_wave_fwd_kernel(const GnP p) {
    constexpr int VEC = VEC16<T>;
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const unsigned lb = xcd_order(blockIdx.x, (unsigned)p.blocks), row_ = lb / (unsigned)p.ncb;
    const int cb = (int)(lb - row_ * p.ncb);
    const long long row = row_, rows = (unsigned)p.blocks / (unsigned)p.ncb;
    const int lv = lane & (p.LV - 1), pos = lane / p.LV, gl = GPV == 1 ? p.Cg / VEC : 1;
    const bool col_ok = cb * p.CB + lv * VEC < p.C;
    const GnLane<T, false> ln(min(cb * p.CB + lv * VEC, p.C - VEC), p.C, 0);
    const int c0 = ln.c0, g0 = c0 / p.Cg;
    const float inv = p.S > 0 ? 1.f / ((float)p.S * (float)p.Cg) : 0.f;
    float ga[VEC], be[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { ga[j] = p.gamma[c0 + j]; be[j] = p.beta[c0 + j]; }
    const auto group_sum = [&](float (&v)[GPV]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < GPV; ++j) {
            for (int o = p.LV; o < 64; o <<= 1) v[j] += __shfl_xor(v[j], o, 64);
            if constexpr (GPV == 1)
                for (int o = 1; o < gl; o <<= 1) v[j] += __shfl_xor(v[j], o, 64);
        }
    };
    for (long long n = row * waves + (threadIdx.x >> 6); n < p.N; n += rows * waves) {
        GnData<T, false> d[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int s = pos + i * p.P;
            d[i].v = make_uint4(0u, 0u, 0u, 0u);
            if (s < p.S) d[i].load(p.x, n * p.xn + s * p.xs + c0, ln);
        }
        GnStat<VEC, GPV> st;
#pragma unroll
        for (int j = 0; j < GPV; ++j) st.m[j] = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            float f[VEC];
            d[i].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) st.m[j * GPV / VEC] += f[j];
            d[i].keep();
        }
        group_sum(st.m);
#pragma unroll
        for (int j = 0; j < GPV; ++j) { st.m[j] *= inv; st.r[j] = 0.f; }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (pos + i * p.P < p.S) {
                float f[VEC];
                d[i].get(f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { const float t = f[j] - st.mean(j); st.r[j * GPV / VEC] = fmaf(t, t, st.r[j * GPV / VEC]); }
            }
            d[i].keep();
        }
        group_sum(st.r);
#pragma unroll
        for (int j = 0; j < GPV; ++j) st.r[j] = 1.f / sqrtf(st.r[j] * inv + p.eps);
        if (col_ok && pos == 0 && (lv & (gl - 1)) == 0) {
#pragma unroll
            for (int j = 0; j < GPV; ++j) { p.mean[n * p.G + g0 + j] = st.m[j]; p.rstd[n * p.G + g0 + j] = st.r[j]; }
        }
        if (p.qo && col_ok) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int s = pos + i * p.P;
                if (s < p.S) {
                    float f[VEC];
                    d[i].get(f);
                    ck_store<VEC>(p, f, n * p.S + s, c0);
                }
                d[i].keep();
            }
        }
        with_act(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int s = pos + i * p.P;
                float f[VEC];
                d[i].get(f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[j] = fmaf((f[j] - st.mean(j)) * st.rstd(j), ga[j], be[j]);
                act_apply<T, decltype(act)::value>(f);
                uint4 o;
                vec_put(o, f);
                if (col_ok && s < p.S) ln.store(p.y, n * p.yn + s * p.ys + c0, o);
            }
        });
    }
}

// ---- workgroup forms -----------------------------------------------------------------------------------------------------
// STATS (chunked): leave (mean, sum of squared distances) of this chunk in part[((n G + g) nchunk + chunk) pieces + piece] and stop.
template <class T, int ITEMS, int GPV, bool TAIL, bool STATS> __global__ __launch_bounds__(GTF, 4) void gn_fwd_kernel(const GnP p) {
    extern __shared__ float lds[];
    constexpr int VEC = VEC16<T>;
    const unsigned lb = xcd_order(STATS ? (unsigned)p.blocks - 1u - blockIdx.x : blockIdx.x, (unsigned)p.blocks);     // (from the back: GnChunk in groupnorm_bwd.h)
    const unsigned t_ = lb / (unsigned)p.ncb, nb_ = STATS ? t_ / (unsigned)p.nchunk : t_;
    const int cb = (int)(lb - t_ * p.ncb), chunk = STATS ? (int)(t_ - nb_ * p.nchunk) : 0;
    const long long nb0 = nb_;
    const GnBlock b = gn_block(p, cb);
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    const int sub = r / p.P, pos = r - sub * p.P;
    const long long n = nb0 * p.NSUB + sub;
    const GnLane<T, TAIL> ln(b.c_lo, b.c_hi, lv);
    const int c0 = ln.c0, col = GPV == 1 ? lv : c0 - b.c_lo;
    const int s_lo = chunk * p.chunk, s_hi = min(p.S, s_lo + p.chunk);
    const bool has = b.c_lo + lv * VEC < b.c_hi, active = sub < p.NSUB && n < p.N && has;
    const auto own = [&](int j) { return has && ln.own(j); };
    float* red = lds;
    float* grp = lds + p.nt * GPV;

    GnData<T, TAIL> d[ITEMS];
    const long long x0 = n * p.xn + (s_lo + pos) * p.xs + c0, y0 = n * p.yn + (s_lo + pos) * p.ys + c0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (active && s_lo + pos + i * p.P < s_hi) d[i].load(p.x, x0 + i * (p.P * p.xs), ln);
    float v[GPV];
#pragma unroll
    for (int j = 0; j < GPV; ++j) v[j] = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (active && s_lo + pos + i * p.P < s_hi) {
            float f[VEC];
            d[i].get(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j * GPV / VEC] += f[j];
            d[i].keep();
        }
    }
    const int cpg = GPV == 1 ? b.cw / VEC : b.cw;
    gn_reduce<GPV>(p, v, red, grp, col, r, b.ng, cpg, own);
    const float inv = s_hi > s_lo ? 1.f / ((float)(s_hi - s_lo) * (float)b.cw) : 0.f;
    GnStat<VEC, GPV> st;
    int gl[GPV];
    group_of<1>(gl, active && p.pieces == 1 ? c0 - b.c_lo : 0, p.Cg, b.ng - 1);       // (an element past a narrow run: any group)
#pragma unroll
    for (int j = 0; j < GPV; ++j) {
        gl[j] = active ? sub * b.ng + gl[j] : 0;
        st.m[j] = grp[gl[j]] * inv;
        v[j] = 0.f;
    }
    float keep_mean = 0.f;                       // a pair's mean, by the thread that stores it
    const int pairs = p.NSUB * b.ng;
    if ((int)threadIdx.x < pairs && pairs <= p.nt) keep_mean = grp[threadIdx.x] * inv;
    if (pairs > p.nt)                             // more pairs than threads: through memory at once (grp is reused below)
        for (int k = threadIdx.x; k < pairs; k += p.nt) {
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
            for (int j = 0; j < VEC; ++j) {
                const float t = f[j] - st.mean(j);
                v[j * GPV / VEC] = fmaf(t, t, v[j * GPV / VEC]);
            }
            d[i].keep();
        }
    }
    gn_reduce<GPV>(p, v, red, grp, col, r, b.ng, cpg, own);
    for (int k = threadIdx.x; k < pairs; k += p.nt) {
        const long long nn = nb0 * p.NSUB + k / b.ng;
        const int g = b.g_lo + k % b.ng;
        if (nn < p.N) {
            if constexpr (STATS) {
                float2* o = p.part + ((nn * p.G + g) * p.nchunk + chunk) * p.pieces + b.piece;
                if (pairs <= p.nt) o->x = keep_mean;
                o->y = grp[k];
            } else {
                if (pairs <= p.nt) p.mean[nn * p.G + g] = keep_mean;
                p.rstd[nn * p.G + g] = 1.f / sqrtf(grp[k] * inv + p.eps);
            }
        }
    }
    if constexpr (!STATS) {
        if (!active) return;
        float ga[VEC], be[VEC];
#pragma unroll
        for (int j = 0; j < GPV; ++j) st.r[j] = 1.f / sqrtf(grp[gl[j]] * inv + p.eps);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int c = TAIL ? min(c0 + j, p.C - 1) : c0 + j;
            ga[j] = p.gamma[c] * st.rstd(j);
            be[j] = p.beta[c];
        }
        if constexpr (!TAIL) {
            if (p.qo) {
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const int s = s_lo + pos + i * p.P;
                    if (s < s_hi) {
                        float f[VEC];
                        d[i].get(f);
                        ck_store<VEC>(p, f, n * p.S + s, c0);
                        d[i].keep();
                    }
                }
            }
        }
        with_act(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int s = s_lo + pos + i * p.P;
                if (s < s_hi) {
                    float f[VEC];
                    d[i].get(f);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] = fmaf(f[j] - st.mean(j), ga[j], be[j]);
                    act_apply<T, decltype(act)::value>(f);
                    uint4 o;
                    vec_put(o, f);
                    ln.store_whole(p.y, y0 + i * (p.P * p.ys), o);
                }
            }
        });
    }
}

// Chunked form, second launch: join the chunks of this block's groups (mean of means, and sums of squared distances moved to it), normalise.
template <class T, int GPV, bool TAIL> __global__ __launch_bounds__(GTF) void gn_apply_kernel(const GnP p) {
    extern __shared__ float lds[];
    constexpr int VEC = VEC16<T>;
    const unsigned lb = xcd_order(blockIdx.x, (unsigned)p.blocks), t_ = lb / (unsigned)p.ncb, n_ = t_ / (unsigned)p.nchunk;
    const int cb = (int)(lb - t_ * p.ncb), chunk = (int)(t_ - n_ * p.nchunk);
    const long long n = n_;
    const GnBlock b = gn_block(p, cb);
    const int parts = p.nchunk * p.pieces;
    float2* stat = (float2*)lds;                 // [ng] (mean, rstd)
    for (int g = threadIdx.x >> 6; g < b.ng; g += p.nt / 64) {
        const float2* a = p.part + (n * p.G + b.g_lo + g) * parts;
        const float m = p.S > 0 ? (float)p.S * (float)p.Cg : 1.f;       // (no positions: both sums are 0, and so are mean and variance)
        const auto count = [&](int i) {
            const int ch = i / p.pieces, pc = i - ch * p.pieces;
            return (float)(min(p.S, (ch + 1) * p.chunk) - ch * p.chunk) * (float)(p.pieces == 1 ? p.Cg : min(p.Cg, (pc + 1) * p.CB) - pc * p.CB);
        };
        float s = 0.f, q = 0.f;
        for (int i = threadIdx.x & 63; i < parts; i += 64) s = fmaf(count(i), a[i].x, s);
        const float mean = wave_total(s) / m;
        for (int i = threadIdx.x & 63; i < parts; i += 64) {
            const float dm = a[i].x - mean;
            q += fmaf(count(i) * dm, dm, a[i].y);
        }
        const float rstd = 1.f / sqrtf(wave_total(q) / m + p.eps);
        if ((threadIdx.x & 63) == 0) {
            stat[g] = make_float2(mean, rstd);
            if (chunk == 0 && b.piece == 0) { p.mean[n * p.G + b.g_lo + g] = mean; p.rstd[n * p.G + b.g_lo + g] = rstd; }
        }
    }
    lds_barrier();
    const int r = (int)threadIdx.x / p.LV, lv = (int)threadIdx.x - r * p.LV;
    if (r >= p.P || b.c_lo + lv * VEC >= b.c_hi) return;
    const GnLane<T, TAIL> ln(b.c_lo, b.c_hi, lv);
    const int c0 = ln.c0;
    GnStat<VEC, GPV> st;
    int gi[GPV];
    group_of<1>(gi, p.pieces == 1 ? c0 - b.c_lo : 0, p.Cg, b.ng - 1);
#pragma unroll
    for (int j = 0; j < GPV; ++j) {
        const float2 t = stat[gi[j]];
        st.m[j] = t.x; st.r[j] = t.y;
    }
    float ga[VEC], be[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int c = TAIL ? min(c0 + j, p.C - 1) : c0 + j;
        ga[j] = p.gamma[c] * st.rstd(j);
        be[j] = p.beta[c];
    }
    const int s_hi = min(p.S, (chunk + 1) * p.chunk);
    with_act(p.act, [&](auto act) __attribute__((always_inline)) {
        for (int s0 = chunk * p.chunk + r; s0 < s_hi; s0 += GU * p.P) {
            GnData<T, TAIL> d[GU];
#pragma unroll
            for (int u = 0; u < GU; ++u)
                if (s0 + u * p.P < s_hi) d[u].load(p.x, n * p.xn + (s0 + u * p.P) * p.xs + c0, ln);
#pragma unroll
            for (int u = 0; u < GU; ++u) {
                const int s = s0 + u * p.P;
                if (s < s_hi) {
                    float f[VEC];
                    d[u].get(f);
                    if constexpr (!TAIL) { if (p.qo) { float t[VEC]; d[u].get(t); ck_store<VEC>(p, t, n * p.S + s, c0); } }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) f[j] = fmaf(f[j] - st.mean(j), ga[j], be[j]);
                    act_apply<T, decltype(act)::value>(f);
                    uint4 o;
                    vec_put(o, f);
                    ln.store(p.y, n * p.yn + s * p.ys + c0, o);
                }
            }
        }
    });
}

// ---- geometry ------------------------------------------------------------------------------------------------------------
int pow2_floor(long long a) { int r = 1; while (2 * r <= a) r *= 2; return r; }

// Whether the kernels of a plan can write the checkpoint with y: a wave's lanes then hold whole blocks of 32 channels.  Widths are multiples of 32,
// and every run of channels starts on one: runs of whole groups begin at a multiple of CB, the pieces of a group wider than a workgroup where
// the group does.
bool ck_in_kernel(const GnP& p, const GnPlan& pl) {
    return !pl.tail && p.C % CK_BLOCK == 0 && p.CB % CK_BLOCK == 0 && (p.pieces == 1 || p.Cg % CK_BLOCK == 0);
}

// even: 16-byte aligned rows
GnPlan gn_plan(GnP& p, int es, bool backward, bool ckpt, bool even) {
    GnPlan pl = {};
    const int vec = 16 / es, GT = backward ? GTB : GTF;
    p.nt = GT;
    const int S = std::max(1, p.S);
    p.pieces = 1; p.nchunk = 1; p.chunk = S; p.NSUB = 1; p.shuf = 0;
    // wave form: groups that are a power of two below a vector, or a power of two of whole vectors
    const int gv = p.Cg % vec == 0 ? p.Cg / vec : 1;                                   // lanes of a group
    if (p.C % vec == 0 && (p.Cg % vec == 0 ? (gv & (gv - 1)) == 0 : vec % p.Cg == 0) && gv <= 64 && p.C / vec >= 2) {
        // as many lanes side by side as the row has, fewer where the positions would not fit
        int lv = std::min(64, pow2_floor(2 * (p.C / vec) - 1));
        while (lv / 2 >= std::max(gv, 2) && (long long)S * lv > 64 * 4 && !(ckpt && lv / 2 * vec < CK_BLOCK)) lv /= 2;
        const int P = 64 / lv, items = cdiv(S, P);
        if (items <= WAVE_ITEMS) {
            pl.form = GN_WAVE;
            pl.items = items;
            pl.gpv = p.Cg % vec == 0 ? 1 : vec / p.Cg;
            p.LV = lv; p.P = P; p.CB = lv * vec; p.ncb = cdiv(p.C, p.CB);
            // 4 waves a workgroup where that leaves every CU one; forward: a wave per sample and channel block (up to 64 rounds), backward:
            // what the chip holds, each leaving a row of column sums
            const int waves = (long long)p.N * p.ncb >= 4 * 256 ? 4 : 1;
            pl.threads = 64 * waves;
            const long long all = cdivll(p.N, waves), cap = std::max<long long>(1, (backward ? 4096 / waves : 32768 / waves) / p.ncb);
            pl.rows = std::min(all, cap);
            pl.blocks = p.blocks = pl.rows * p.ncb;
            pl.part = backward ? (size_t)pl.rows * p.C : 0;
            return pl;
        }
    }
    const bool gs = p.Cg % vec == 0;
    // whole groups that start on the vector grid; where rows do not end on it anyway, any whole groups
    long long unit = p.C % vec ? p.Cg : std::lcm((long long)p.Cg, (long long)vec);
    pl.gpv = gs ? 1 : vec;
    // piped form (backward): 32 lanes or fewer side by side (a power of two), at most 8 vectors a thread
    if (backward && even && p.C % vec == 0 && unit <= 32 * vec) {
        const auto fits = [&](int lv) { return (lv * vec) % unit == 0 && lv / 2 * vec < p.C && cdiv(S, GTP / lv) <= PIPED_ITEMS && S >= GTP / lv; };
        int lv = 32;
        while (lv > 1 && !fits(lv)) lv /= 2;
        while (lv > 4 && cdiv(S, GTP / lv) > 4 && (long long)p.N * cdiv(p.C, lv * vec) < 1024 && fits(lv / 2)) lv /= 2;
        if (lv > 1 && (long long)p.N * cdiv(p.C, lv * vec) >= 512) {
            pl.form = GN_PIPED;
            pl.gpv = gs ? 1 : vec / p.Cg;                            // (unit is vec times a power of two: so is Cg, or it divides vec)
            p.LV = lv; p.P = GTP / lv; p.CB = lv * vec; p.ncb = cdiv(p.C, p.CB);
            pl.threads = GTP;
            pl.rows = std::min<long long>(p.N, std::max(1, 256 / p.ncb));
            pl.blocks = p.blocks = pl.rows * p.ncb;
            pl.part = (size_t)pl.rows * p.C;
            return pl;
        }
    }
    const int cap = GT * vec;
    if (unit > cap) unit = p.Cg;
    if (unit > cap) {                                       // a group wider than a workgroup's lanes
        p.CB = cap;
        p.pieces = cdiv(p.Cg, cap);
        p.ncb = p.G * p.pieces;
        pl.tail = p.Cg % vec != 0;
    } else {
        // at least 128 bytes of a position side by side (a cache line), and enough channels for every thread where S is short
        const long long want = std::max<long long>(128 / es, (long long)GT * vec / S);
        long long cb = unit;
        while (cb * 2 <= cap && cb < want && cb < p.C) cb *= 2;
        p.CB = (int)std::min<long long>(cb, p.C);
        p.ncb = cdiv(p.C, p.CB);
        pl.tail = p.C % vec != 0 || unit % vec != 0;
    }
    // off the grid: blocks of nearly equal numbers of groups, the last one a whole vector wide too
    const auto even_out = [&]() {
        if (!pl.tail || p.pieces > 1) return;
        int per = cdiv(p.G, cdiv(p.G, p.CB / p.Cg));
        const auto thin = [&]() { return per < p.G && (p.G - (cdiv(p.G, per) - 1) * per) * p.Cg < vec; };
        while (thin() && (per + 1) * p.Cg <= cap) ++per;
        while (thin() && per > 1) --per;
        p.CB = per * p.Cg;
        p.ncb = cdiv(p.G, per);
    };
    even_out();
    const auto lanes = [&]() {
        p.LV = cdiv(p.CB, vec);
        p.P = p.nt / p.LV;
        p.NSUB = 1;
        if (p.P > S) { p.P = S; p.NSUB = std::min(p.nt / (p.LV * p.P), std::max(1, p.N)); }
        p.shuf = p.NSUB == 1 && p.LV <= 32 && (p.LV & (p.LV - 1)) == 0 && p.P * p.LV == p.nt;
    };
    lanes();
    // fewer channels side by side, down to 32 bytes, where a run of groups does not fit a workgroup's registers or where there would be fewer
    // workgroups than CUs (the blocks that share a cache line run on one XCD).  Forward, 32 bytes so and chunked: 64, 512 x 4096 x 64 bf16 23, 185 us
    // and 28, 199; 64 x 4096 x 64 fp32 36 and 44.  fp32 that passes the 256 MB cache is the other way round (512 x 4096 x 64 349 and 311, x 128 679
    // and 587): down to 64 bytes there.
    const int narrow = es == 4 && (long long)p.N * S * p.C * es >= 1LL << 28 ? 64 : 32;
    const auto halves = [&]() { return pl.tail ? p.CB > p.Cg && cdiv(p.CB / p.Cg, 2) * p.Cg * es >= narrow
                                               : p.CB % 2 == 0 && (p.CB / 2) % unit == 0 && p.CB / 2 * es >= narrow && !(ckpt && p.CB % 64); };
    while (p.pieces == 1 && halves() &&
           (cdiv(S, p.P) > ITEMS_MAX || (S * (long long)p.CB > 16 * vec * 64 && cdivll(p.N, p.NSUB) * p.ncb < 512))) {
        const int before = p.CB;
        p.CB = pl.tail ? cdiv(p.CB / p.Cg, 2) * p.Cg : p.CB / 2;
        p.ncb = cdiv(p.C, p.CB);
        even_out();
        lanes();
        if (p.CB == before) break;
    }
    // forward, vectors of several groups: what a thread does besides its vectors costs as much as some 8 of them, so smaller workgroups of up to 8
    // vectors a thread while the chip keeps 4 waves a CU (300 x 50 x 231 bf16: 14 us, 23 with 512 threads; not with one group a vector, 64 x 1024 x
    // 64: 12.5 and 9.6, nor backward, 300 x 50 x 231 fp32: 26 and 24)
    while (!backward && !gs && p.pieces == 1 && p.nt > 64 && p.nt / 2 >= p.LV) {
        const GnP before = p;
        p.nt /= 2;
        lanes();
        if (cdiv(S, p.P) > 8 || cdivll(p.N, p.NSUB) * p.ncb * (p.nt / 64) < 1024) { p = before; break; }
    }
    const long long held_blocks = cdivll(p.N, p.NSUB) * p.ncb;
    // held with fewer workgroups than CUs, and chunked: 64 of them (8 x 4096 x 64 fp32, 16 x 4096 x 64 bf16) 18.1, 17.7 us and 14.4, 14.1; 192 (24 x 4096 x 64
    // fp32) 23.3 and 28.8; 64 and 100 off the grid (64 x 1000 x 33, 100 x 1500 x 15 bf16) 14.0, 13.6 and 19.9, 18.2.  With a checkpoint, whose runs are 32
    // channels wide at least (halves()) and so twice as long a thread: 96 (48 x 2048 x 64 bf16) 23.9 and 20.0, 128 (64 x 1024 x 64 bf16, fp32) 16.7, 25.9 and
    // 15.6, 22.6; 192 (24 x 512 x 256 fp32) 16.8 and 20.2, 200 (200 x 1500 x 32 bf16) 23.2 and 28.9
    if (p.pieces == 1 && cdiv(S, p.P) <= ITEMS_MAX && (held_blocks >= (ckpt ? 160 : pl.tail ? 64 : 96) || cdiv(S, p.P) <= 4)) {
        pl.form = GN_HELD;
        pl.items = cdiv(S, p.P);
        // backward: a workgroup goes over several samples and leaves one row of column sums
        pl.rows = backward ? std::min<long long>(cdivll(p.N, p.NSUB), std::max(1, 2048 / p.ncb)) : 0;
        pl.blocks = backward ? pl.rows * p.ncb : held_blocks;
        pl.part = backward ? (size_t)pl.rows * p.C : 0;
    } else {
        pl.form = GN_CHUNKED;
        while (p.pieces == 1 && p.CB * es < 128 && p.CB * 2 <= std::min(cap, p.C)) p.CB *= 2;   // whole cache lines again
        if (p.pieces == 1) { p.ncb = cdiv(p.C, p.CB); even_out(); p.LV = cdiv(p.CB, vec); }
        p.NSUB = 1;
        p.nt = GT;
        p.P = std::max(1, GT / p.LV);
        p.shuf = p.LV <= 32 && (p.LV & (p.LV - 1)) == 0 && p.P * p.LV == GT;
        pl.items = ITEMS_MAX;
        // forward: chunks of what a workgroup holds, shorter where that leaves the chip empty; backward: about 2048 workgroups
        long long chunk = backward ? cdivll(cdivll((long long)p.N * p.ncb * S, 2048), GU * p.P) * GU * p.P : (long long)p.P * ITEMS_MAX;
        while (chunk > GU * p.P && (long long)p.N * p.ncb * cdivll(S, chunk) < 512) chunk = cdivll(chunk / 2, p.P) * p.P;
        p.chunk = (int)std::max<long long>(1, std::min<long long>(chunk, S));          // (an empty batch has chunks too)
        p.nchunk = cdiv(S, p.chunk);
        pl.blocks = (long long)p.N * p.ncb * p.nchunk;
        pl.rows = (long long)p.N * p.nchunk;
        pl.part = backward ? (size_t)pl.rows * p.C + (size_t)p.N * p.G : (size_t)p.N * p.G * p.nchunk * p.pieces;
    }
    pl.threads = p.nt;
    p.blocks = pl.blocks;
    return pl;
}

template <class T> int gn_fwd(const GnP& p, const GnPlan& pl, hipStream_t st) {
    if (pl.form == GN_WAVE)
        return gn_wave_variants<T>(pl, [&](auto gpv, auto items) {
            return gn_launch(gn_wave_fwd_kernel<T, decltype(items)::value, decltype(gpv)::value>, p, pl.threads, 0, st);
        });
    return gn_variants<T>(pl, [&](auto gpv, auto tail) {
        constexpr int GPV = decltype(gpv)::value;
        constexpr bool TAIL = decltype(tail)::value;
        const int gpb = cdiv(p.CB, std::min(p.Cg, p.CB));
        const size_t lds = sizeof(float) * ((size_t)p.nt * GPV + (size_t)p.NSUB * (gpb + (p.shuf ? 0 : p.LV * GPV)));
        if (pl.form == GN_HELD)
            return pl.items <= 4 ? gn_launch(gn_fwd_kernel<T, 4, GPV, TAIL, false>, p, p.nt, lds, st)
                                 : gn_launch(gn_fwd_kernel<T, ITEMS_MAX, GPV, TAIL, false>, p, p.nt, lds, st);
        const int rc = gn_launch(gn_fwd_kernel<T, ITEMS_MAX, GPV, TAIL, true>, p, p.nt, lds, st);
        if (rc != FAVAE_OK) return rc;
        return gn_launch(gn_apply_kernel<T, GPV, TAIL>, p, p.nt, sizeof(float2) * gpb, st);
    });
}

int gn_sizes(const char* who, long long N, long long S, int C, int G, int act, int dtype) {
    FAVAE_CHECK_ARG(dtype == FAVAE_F32 || dtype == FAVAE_BF16, "%s: dtype is neither fp32 nor bf16", who);
    FAVAE_CHECK_ARG(act >= FAVAE_ACT_NONE && act <= FAVAE_ACT_GELU_TANH, "%s: unknown activation %d", who, act);
    FAVAE_CHECK_ARG(N >= 0 && S >= 0 && C >= 1 && G >= 1 && C % G == 0, "%s: C = %d channels do not divide into G = %d groups, or a negative size", who, C, G);
    FAVAE_CHECK_ARG(N <= 0x7fffffff && S <= 0x3fffffff && N * S <= (1LL << 38) && C <= (1 << 24), "%s: N, S or C too large", who);
    return FAVAE_OK;
}
// limits of the launches, checked before the first of them
int gn_fits(const char* who, const GnP& p, const GnPlan& pl, size_t scratch_bytes) {
    FAVAE_CHECK_ARG(pl.blocks <= 0x7fffffffLL, "%s: too many samples for one launch", who);
    FAVAE_CHECK_ARG(pl.form != GN_CHUNKED || (long long)p.N * p.G <= 0x7fffffffLL, "%s: too many groups for one launch", who);
    FAVAE_CHECK_ARG(pl.part * sizeof(float2) <= scratch_bytes && (pl.part == 0 || p.part), "%s: scratch of %zu bytes, %zu needed", who, scratch_bytes,
                    pl.part * sizeof(float2));
    return FAVAE_OK;
}
bool aligned(const void* a, int es) { return (uintptr_t)a % (size_t)es == 0; }
// 16-byte aligned rows, and a sample within 31 bits
bool even16(const void* a, long long n, long long s, long long S, int C, int es) {
    return aligned(a, 16) && n * es % 16 == 0 && s * es % 16 == 0 && (S * s + C) * es < 0x70000000LL;
}

}  // namespace

extern "C" size_t favae_gn_act_scratch(long long N, long long S, int C, int G, int backward, int dtype) {
    if (gn_sizes("favae_gn_act_scratch", N, S, C, G, FAVAE_ACT_NONE, dtype) != FAVAE_OK) return 0;
    size_t need = 0;
    for (bool either : {false, true}) {                     // forward: with a checkpoint or without; backward: aligned or not
        GnP p = {};
        p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G;
        need = std::max(need, gn_plan(p, dtype == FAVAE_F32 ? 4 : 2, backward != 0, either && !backward, either && backward).part);
    }
    return need * sizeof(float2);
}

extern "C" int favae_debug_gn_act_plan(long long N, long long S, int C, int G, int backward, int either, int dtype, int* out12) {
    const int rc = gn_sizes("favae_debug_gn_act_plan", N, S, C, G, FAVAE_ACT_NONE, dtype);
    if (rc != FAVAE_OK) return rc;
    FAVAE_CHECK_ARG(out12, "favae_debug_gn_act_plan: null pointer");
    GnP p = {};
    p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G;
    const GnPlan pl = gn_plan(p, dtype == FAVAE_F32 ? 4 : 2, backward != 0, !backward && either && C % CK_BLOCK == 0, backward && either);
    const int v[12] = {pl.form, pl.items, pl.gpv, pl.tail, p.pieces, p.NSUB, p.P, p.ncb, p.nchunk, p.CB, (int)std::min<long long>(pl.rows, 0x7fffffff), ck_in_kernel(p, pl)};
    std::copy(v, v + 12, out12);
    return FAVAE_OK;
}

extern "C" int favae_gn_act_fwd(const void* x, long long xn, long long xs, long long N, long long S, int C, int G, const float* gamma,
                                const float* beta, float eps, int act, void* y, long long yn, long long ys, float* mean, float* rstd,
                                void* q, void* e, void* scratch, size_t scratch_bytes, int dtype, void* stream) {
    const int rc = gn_sizes("favae_gn_act_fwd", N, S, C, G, act, dtype);
    if (rc != FAVAE_OK) return rc;
    if (N == 0) return FAVAE_OK;
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(gamma && beta && mean && rstd && (S == 0 || (x && y)), "favae_gn_act_fwd: null pointer");
    FAVAE_CHECK_ARG((q != nullptr) == (e != nullptr), "favae_gn_act_fwd: q and e, or neither");
    FAVAE_CHECK_ARG(S <= 1 || (xs >= C && ys >= C), "favae_gn_act_fwd: a position's stride is below C");
    FAVAE_CHECK_ARG(aligned(x, es) && aligned(y, es), "favae_gn_act_fwd: a pointer is not aligned to its type");
    GnP p = {};
    p.x = x; p.xn = xn; p.xs = xs; p.y = y; p.yn = yn; p.ys = ys;
    p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd; p.part = (float2*)scratch;
    p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G; p.act = act; p.eps = eps; p.nb = cdiv(C, CK_BLOCK);
    const GnPlan pl = gn_plan(p, es, false, q && C % CK_BLOCK == 0, false);       // (other widths are packed in a launch of their own)
    const int fit = gn_fits("favae_gn_act_fwd", p, pl, scratch_bytes);
    if (fit != FAVAE_OK) return fit;
    if (q && S > 0) {
        // the checkpoint leaves with y, or in a launch of its own first
        if (ck_in_kernel(p, pl)) {
            p.qo = (unsigned char*)q;
            p.eo = (unsigned char*)e;
        } else {
            const int r2 = ck_pack_samples(x, xn, xs, N, S, C, q, C, e, p.nb, dtype, (hipStream_t)stream);
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
    const bool any = N > 0 && S > 0;
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(gamma && beta && (!any || (dy && dx && mean && rstd)), "favae_gn_act_bwd: null pointer");
    FAVAE_CHECK_ARG(!any || (x != nullptr) != (q != nullptr && e != nullptr), "favae_gn_act_bwd: x, or its 8-bit checkpoint (q and e), and not both");
    FAVAE_CHECK_ARG(S <= 1 || (ds >= C && dxs >= C && (!x || xs >= C)), "favae_gn_act_bwd: a position's stride is below C");
    FAVAE_CHECK_ARG(aligned(x, es) && aligned(dy, es) && aligned(dx, es), "favae_gn_act_bwd: a pointer is not aligned to its type");
    GnP p = {};
    p.x = x; p.xn = xn; p.xs = xs; p.q = (const unsigned char*)q; p.e = (const unsigned char*)e; p.dy = dy; p.dn = dn; p.ds = ds;
    p.y = dx; p.yn = dxn; p.ys = dxs;
    p.gamma = gamma; p.beta = beta; p.mean = (float*)mean; p.rstd = (float*)rstd; p.part = (float2*)scratch;
    p.N = (int)N; p.S = (int)S; p.C = C; p.G = G; p.Cg = C / G; p.act = act; p.nb = cdiv(C, CK_BLOCK);
    GnPlan pl = {};
    if (any) {
        const bool even = (!x || even16(x, xn, xs, S, C, es)) && even16(dy, dn, ds, S, C, es) && even16(dx, dxn, dxs, S, C, es);
        pl = gn_plan(p, es, true, false, even);
        const int fit = gn_fits("favae_gn_act_bwd", p, pl, scratch_bytes);
        if (fit != FAVAE_OK) return fit;
        p.s12 = p.part + (size_t)pl.rows * C;
    }
    return dtype == FAVAE_F32 ? gn_bwd_f32(p, pl, dgamma, dbeta, (hipStream_t)stream) : gn_bwd_bf16(p, pl, dgamma, dbeta, (hipStream_t)stream);
}
