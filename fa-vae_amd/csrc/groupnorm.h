// Group norm with an activation: what its forward (groupnorm.hip) and backward (groupnorm_bwd.h) kernels share.
#pragma once
#include "act8.h"
#include <algorithm>
#include <type_traits>

constexpr int GTF = 512, GTB = 256;     // threads of a workgroup, forward and backward, at most
constexpr int GU = 4;                   // positions a thread has under way in the chunked forms
constexpr int WAVE_ITEMS = 8, ITEMS_MAX = 16;
constexpr int GTP = 512, PIPED_ITEMS = 8;        // piped form

enum GnForm { GN_WAVE, GN_PIPED, GN_HELD, GN_CHUNKED };

struct GnP {
    const void *x, *dy;
    void* y;                            // y, or dx
    const unsigned char *q, *e;         // x as an 8-bit checkpoint, [N][S][C] and [N][S][nb]
    unsigned char *qo, *eo;             // forward: the same, to be written, or NULL
    long long xn, xs, dn, ds, yn, ys;   // strides of a sample and of a position, in elements
    const float *gamma, *beta;
    float *mean, *rstd;                 // [N][G]
    float2* part;                       // partial sums, see the kernels
    float2* s12;                        // chunked backward: (s1, s2) / m of every group, [N][G]
    int N, S, C, G, Cg, act, nb;
    float eps;
    // geometry.  A workgroup (a wave in the wave form) takes CB channels: whole groups (pieces == 1), or piece j of `pieces` of one group
    // wider than it.  LV lanes side by side, 16 bytes each, cover the CB channels, P rows of lanes take P positions at once, NSUB samples share a
    // workgroup.
    int LV, P, NSUB, CB, ncb, pieces, chunk, nchunk, shuf, nt;      // nt: threads
    long long blocks;
};

struct GnPlan {
    GnForm form;
    int items, gpv;                     // 16-byte vectors a thread holds; groups a vector may touch (VEC: any)
    bool tail;                          // a run of channels may end inside a vector, or start off the vector grid
    int threads;
    long long blocks, rows;             // rows of column sums (backward)
    size_t part;                        // float2 entries of workspace
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
__device__ __forceinline__ unsigned xcd_order(unsigned b, unsigned n) {
    const unsigned per = n / 8;
    return b < per * 8 ? (b & 7) * per + (b >> 3) : b;
}
// groups of elements c, c + STEP, ... (counted from a group's start), at most `last`; STEP <= Cg.  Divisions are 32 bits wide and few: a 64-bit
// one is 100 to 150 instructions.
template <int STEP, int N> __device__ __forceinline__ void group_of(int (&g)[N], int c, int Cg, int last) {
    int q = c / Cg, r = c - q * Cg;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        g[j] = min(q, last);
        r += STEP;
        if (r >= Cg) { r -= Cg; ++q; }
    }
}

// barrier for data in LDS: vector memory operations stay under way (__syncthreads waits for them)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// log2 of the lanes (up to 64) that add the `per` values of each of `pairs` sums side by side
__device__ __forceinline__ int pair_lanes_log2(int threads, int pairs, int per) {
    int s = 6;
    while (s > 0 && (pairs << s > threads || 1 << (s - 1) >= per)) --s;
    return s;
}

// Sum of v over the threads of every (sample of the block, group of the block) pair into grp[].  A thread's values j with own(j) belong
// to columns col + j of its row; a group is cpg neighbouring columns.  With p.shuf the 64 / LV rows of a wave are added by
// shuffles first.  Every thread of the block calls; values of idle threads are 0.
template <int NV, class O>
__device__ __forceinline__ void gn_reduce(const GnP& p, float (&v)[NV], float* red, float* grp, int col, int r, int ng, int cpg, O&& own) {
    const int cols = p.LV * NV;
    int rows = p.P;
    if (p.shuf) {
        for (int o = p.LV; o < 64; o <<= 1)
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] += __shfl_xor(v[j], o, 64);
        rows = p.nt / 64;
        if ((int)(threadIdx.x & 63) < p.LV)
#pragma unroll
            for (int j = 0; j < NV; ++j) if (own(j)) red[(threadIdx.x >> 6) * cols + col + j] = v[j];
    } else if (r < p.P * p.NSUB) {
#pragma unroll
        for (int j = 0; j < NV; ++j) if (own(j)) red[r * cols + col + j] = v[j];
    }
    lds_barrier();
    const int pairs = p.NSUB * ng;
    if (!p.shuf) {
        // many rows: the columns first (with a division for each value, and partial vectors stored element by element, 512 x 195 x 210 bf16 took 45 us, now 41)
        const int all = p.NSUB * cols, ls = pair_lanes_log2(p.nt, all, rows), L = 1 << ls, l = (int)threadIdx.x & (L - 1);
        float* tot = grp + pairs;
        for (int k = (int)threadIdx.x >> ls; k < all; k += p.nt >> ls) {
            const int sub = k / cols;
            const float* a = red + (sub * rows + l) * cols + k - sub * cols;
            float s = 0.f;
            for (int i = l; i < rows; i += L) { s += *a; a += L * cols; }
            for (int o = L >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            if (l == 0) tot[k] = s;
        }
        lds_barrier();
        red = tot;
        rows = 1;
    }
    // L lanes take a pair: as many as there are threads for every pair at once, at most its values
    const int per = rows * cpg, ls = pair_lanes_log2(p.nt, pairs, per), L = 1 << ls, l = (int)threadIdx.x & (L - 1);
    for (int k = (int)threadIdx.x >> ls; k < pairs; k += p.nt >> ls) {
        const int sub = k / ng, g = k - sub * ng;
        float s = 0.f;
        for (int i = l; i < per; i += L) {
            const int row = rows == 1 ? 0 : i / cpg, c = i - row * cpg;
            s += red[(sub * rows + row) * cols + g * cpg + c];
        }
        for (int o = L >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (l == 0) grp[k] = s;
    }
    lds_barrier();
}

// The values a thread holds are kept as they lie in memory and converted anew in every pass: without this the compiler keeps the fp32
// values of the first pass for the next, twice the registers
__device__ __forceinline__ void hold(uint4& r) { asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); }
__device__ __forceinline__ void hold(unsigned& r) { asm volatile("" : "+v"(r)); }
__device__ __forceinline__ void hold(float& r) { asm volatile("" : "+v"(r)); }

// A thread's channels: the vector from c0 on, of which elements j_lo .. j_hi - 1 are its own.  The last vector of a run that does not end on
// the vector grid starts early, so that it is whole (its first elements then belong to the lane before it); a run narrower than a vector
// is loaded element by element.
template <class T, bool TAIL> struct GnLane {
    static constexpr int VEC = VEC16<T>;
    int c0, j_lo, j_hi;
    __device__ __forceinline__ GnLane(int c_lo, int c_hi, int lv) {
        c0 = c_lo + lv * VEC; j_lo = 0; j_hi = VEC;
        if constexpr (TAIL) {
            if (c_hi - c_lo < VEC) j_hi = c_hi - c_lo;
            else if (c0 + VEC > c_hi) { j_lo = c0 - (c_hi - VEC); c0 = c_hi - VEC; }
        }
    }
    __device__ __forceinline__ bool own(int j) const { return !TAIL || (j >= j_lo && j < j_hi); }
    // the whole vector, with the elements that the lane before writes too, to the same values: where every thread of the block has read
    // what it needs (`out` may be the input)
    __device__ __forceinline__ void store_whole(void* base, long long off, const uint4& r) const { store16((T*)base + off, r, TAIL ? j_hi : VEC); }
    __device__ __forceinline__ void store(void* base, long long off, const uint4& r) const {
        T* a = (T*)base + off;
        if (!TAIL || j_hi - j_lo == VEC) __builtin_memcpy(a, &r, 16);
        else {
            T t[VEC];
            __builtin_memcpy(t, &r, 16);
#pragma unroll
            for (int j = 0; j < VEC; ++j) if (own(j)) a[j] = t[j];
        }
    }
};
// A vector of a tensor
template <class T, bool TAIL> struct GnData {
    static constexpr int VEC = VEC16<T>;
    uint4 v;
    __device__ __forceinline__ void load(const void* base, long long off, const GnLane<T, TAIL>& l) { v = load16((const T*)base + off, TAIL ? l.j_hi : VEC); }
    __device__ __forceinline__ void get(float (&f)[VEC]) const { vec_get(f, v); }
    __device__ __forceinline__ void keep() { hold(v); }
};
// The same of an 8-bit checkpoint.  Without TAIL it lies inside one block of 32 channels, with it the elements from k0 on belong to the next.
template <class T, bool TAIL> struct CkData {
    static constexpr int VEC = VEC16<T>;
    unsigned w[VEC / 4];
    float s, s1;
    int k0;
    __device__ __forceinline__ void load(const unsigned char* q, const unsigned char* e, long long pos, int C, int nb, const GnLane<T, TAIL>& l) {
        const unsigned char* a = q + pos * C + l.c0;
        e += pos * nb + (l.c0 >> 5);
        s = ck_scale(e[0]);
        if constexpr (!TAIL) __builtin_memcpy(w, a, VEC);
        else {
            k0 = 32 - (l.c0 & 31);
            s1 = ck_scale(e[k0 < l.j_hi ? 1 : 0]);
            if (l.j_hi == VEC) __builtin_memcpy(w, a, VEC);
            else {
#pragma unroll
                for (int j = 0; j < VEC / 4; ++j) w[j] = 0u;
#pragma unroll
                for (int j = 0; j < VEC; ++j) if (j < l.j_hi) w[j >> 2] |= (unsigned)a[j] << (8 * (j & 3));
            }
        }
    }
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = ck_value(w[j >> 2], j & 3, TAIL && j >= k0 ? s1 : s);
    }
    __device__ __forceinline__ void keep() {
#pragma unroll
        for (int j = 0; j < VEC / 4; ++j) hold(w[j]);
        hold(s);
    }
};

// ---- piped form: 16 bytes a lane between memory and LDS or registers through a buffer descriptor of one sample ---------------
typedef unsigned gn_v4u __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* gn_lds;
constexpr unsigned GN_NOWHERE = 0x80000000u;         // an offset outside every descriptor: loads give zeros, stores are dropped
__device__ __forceinline__ __amdgpu_buffer_rsrc_t gn_rsrc(const void* base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + bytes), 0, 0x7fffffff, 0x00020000);
}
// items of a sample into buf[item][thread]: first offset `off`, `step` bytes between items, the first `mine` of them exist
template <int ITEMS> __device__ __forceinline__ void gn_dma(char* buf, int wave, const __amdgpu_buffer_rsrc_t r, unsigned off, unsigned step, int mine) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (gn_lds)(buf + (i * GTP + wave * 64) * 16), 16, (int)(i < mine ? off + i * step : GN_NOWHERE), 0, 0, 0);
}

// Mean and rstd of a thread's channels: GPV values a vector, VEC / GPV neighbouring channels each
template <int VEC, int GPV> struct GnStat {
    float m[GPV], r[GPV];
    __device__ __forceinline__ float mean(int j) const { return m[j * GPV / VEC]; }
    __device__ __forceinline__ float rstd(int j) const { return r[j * GPV / VEC]; }
};

// f(integral_constant<GPV>, bool_constant<TAIL>) for the workgroup forms, where a vector touches one group or any
template <class T, class F> int gn_variants(const GnPlan& pl, F&& f) {
    if (pl.gpv == 1) return f(std::integral_constant<int, 1>(), std::false_type());
    if (!pl.tail) return f(std::integral_constant<int, VEC16<T>>(), std::false_type());
    return f(std::integral_constant<int, VEC16<T>>(), std::true_type());
}
// f(integral_constant<GPV>)
template <class T, class F> int gn_gpv(const GnPlan& pl, F&& f) {
    if (pl.gpv == 1) return f(std::integral_constant<int, 1>());
    if (pl.gpv == 2) return f(std::integral_constant<int, 2>());
    if (pl.gpv == 4) return f(std::integral_constant<int, 4>());
    return f(std::integral_constant<int, VEC16<T>>());
}
// f(integral_constant<GPV>, integral_constant<ITEMS>) for the wave form
template <class T, class F> int gn_wave_variants(const GnPlan& pl, F&& f) {
    const auto items = [&](auto gpv) {
        if (pl.items <= 1) return f(gpv, std::integral_constant<int, 1>());
        if (pl.items <= 2) return f(gpv, std::integral_constant<int, 2>());
        if (pl.items <= 4) return f(gpv, std::integral_constant<int, 4>());
        return f(gpv, std::integral_constant<int, WAVE_ITEMS>());
    };
    return gn_gpv<T>(pl, items);
}

template <class K> int gn_launch(K k, const GnP& p, int threads, size_t lds, hipStream_t st) {
    if (p.blocks > 0) k<<<(unsigned)p.blocks, threads, lds, st>>>(p);
    FAVAE_LAUNCH_CHECK();
    return FAVAE_OK;
}

// backward kernels, one translation unit per type (gn_bwd_f32.hip, gn_bwd_bf16.hip); dgamma and dbeta may be NULL
int gn_bwd_f32(const GnP& p, const GnPlan& pl, float* dgamma, float* dbeta, hipStream_t st);
int gn_bwd_bf16(const GnP& p, const GnPlan& pl, float* dgamma, float* dbeta, hipStream_t st);
