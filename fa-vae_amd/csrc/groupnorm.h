// Group norm with an activation: what its forward (groupnorm.hip) and backward (groupnorm_bwd.h) kernels share.
#pragma once
#include "act8.h"
#include <algorithm>
#include <type_traits>


constexpr int GTF = 512, GTB = 256;     // threads of a workgroup, forward and backward
constexpr int U = 4;                    // positions a thread has under way in the chunked form's second pass

struct GnP {
    const void *x, *dy;
    void* y;                            // y, or dx
    const unsigned char *q, *e;         // x as an 8-bit checkpoint, [N][S][C] and [N][S][nb]
    unsigned char *qo, *eo;             // forward: the same, to be written, or NULL
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

constexpr int ITEMS_MAX = 16;
struct GnPlan { int vec; bool gs, held; int items; long long blocks; size_t part; };   // part: float2 entries of workspace

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

// lanes (a power of two up to 64) that add the `per` values of each of `pairs` sums side by side
template <int GT> __device__ __forceinline__ int pair_lanes(int pairs, int per) {
    int L = 64;
    while (L > 1 && (pairs * L > GT || L / 2 >= per)) L >>= 1;
    return L;
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
        rows = GTF / 64;
        if ((int)(threadIdx.x & 63) < p.LV)
#pragma unroll
            for (int j = 0; j < NV; ++j) red[(threadIdx.x >> 6) * cols + lv * NV + j] = v[j];
    } else if (r < p.P * p.NSUB) {
#pragma unroll
        for (int j = 0; j < NV; ++j) red[r * cols + lv * NV + j] = v[j];
    }
    __syncthreads();
    // L lanes take a pair: as many as there are threads for every pair at once, at most its values
    const int pairs = p.NSUB * ng, per = rows * cpg, L = pair_lanes<GTF>(pairs, per), l = (int)threadIdx.x & (L - 1);
    for (int k = (int)threadIdx.x / L; k < pairs; k += GTF / L) {
        const int sub = k / ng, g = k - sub * ng;
        float s = 0.f;
        for (int i = l; i < per; i += L) {
            const int row = i / cpg, c = i - row * cpg;
            s += red[(sub * rows + row) * cols + g * cpg + c];
        }
        for (int o = L >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (l == 0) grp[k] = s;
    }
    __syncthreads();
}

// The values a thread holds are kept as they lie in memory and converted anew in every pass: without this the compiler keeps the fp32
// values of the first pass for the next, twice the registers
__device__ __forceinline__ void hold(uint4& r) { asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); }
__device__ __forceinline__ void hold(float4& r) { asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); }
__device__ __forceinline__ void hold(float2& r) { asm volatile("" : "+v"(r.x), "+v"(r.y)); }
__device__ __forceinline__ void hold(unsigned& r) { asm volatile("" : "+v"(r)); }
__device__ __forceinline__ void hold(float& r) { asm volatile("" : "+v"(r)); }
__device__ __forceinline__ void hold(bf16_t& r) { asm volatile("" : "+v"(r)); }

template <class T, int VEC> struct GnData {
    typedef typename VecOf<T, VEC>::raw raw;
    raw v;
    __device__ __forceinline__ void load(const void* base, long long off) { v = *(const raw*)((const T*)base + off); }
    __device__ __forceinline__ void get(float (&f)[VEC]) const { vec_get(f, v); }
    __device__ __forceinline__ void keep() { hold(v); }
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
    __device__ __forceinline__ void keep() {
        hold(w[0]);
        if constexpr (VEC == 8) hold(w[1]);
        hold(s);
    }
};

// VEC values of a position into an 8-bit checkpoint: 32 / VEC neighbouring lanes hold a block (C a multiple of 32, all of them active)
template <int VEC> __device__ __forceinline__ void ck_store(const GnP& p, const float (&f)[VEC], long long pos, int c) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 32 / VEC; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    const unsigned code = ck_code(m);
    unsigned w[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[j >> 2] |= ((unsigned)ck_round(f[j], code) & 0xffu) << (8 * (j & 3));
    unsigned char* o = p.qo + pos * p.C + c;
    if constexpr (VEC == 8) *(uint2*)o = make_uint2(w[0], w[1]);
    else *(unsigned*)o = w[0];
    if ((c & 31) == 0) p.eo[pos * p.nb + (c >> 5)] = (unsigned char)code;
}

// Per-channel constants of a thread.  GS: a vector lies inside one group, so that its mean and rstd are single values.
template <int VEC, bool GS> struct GnStat {
    float m[GS ? 1 : VEC], r[GS ? 1 : VEC];
    __device__ __forceinline__ float mean(int j) const { return m[GS ? 0 : j]; }
    __device__ __forceinline__ float rstd(int j) const { return r[GS ? 0 : j]; }
};

#define GN_VEC(T, vec, F)                                                              \
    do {                                                                               \
        if constexpr (sizeof(T) == 4) { if ((vec) == 4) F(T, 4) else if ((vec) == 2) F(T, 2) else F(T, 1) } \
        else { if ((vec) == 8) F(T, 8) else if ((vec) == 2) F(T, 2) else F(T, 1) }     \
    } while (0)

template <class K> int gn_launch(K k, const GnP& p, int threads, size_t lds, hipStream_t st) {
    FAVAE_CHECK_ARG(p.blocks <= 0x7fffffffLL, "favae_gn_act: too many samples for one launch");
    if (p.blocks > 0) k<<<(unsigned)p.blocks, threads, lds, st>>>(p);
    FAVAE_LAUNCH_CHECK();
    return FAVAE_OK;
}

// backward kernels, one translation unit per type (gn_bwd_f32.hip, gn_bwd_bf16.hip)
int gn_bwd_f32(const GnP& p, const GnPlan& pl, hipStream_t st);
int gn_bwd_bf16(const GnP& p, const GnPlan& pl, hipStream_t st);
