// Matrix product with bias, activation and residual in its epilogue, forward and backward.
//
//   forward    u = x w^T + bias,  y = act(u) + residual                       x [M][K], w [N][K]
//   backward   du = dy act'(u),  dx = du w,  dw = du^T x,  db = column sums of du
//
// All three products are out[i][j] = sum_c P(i, c) Q(j, c).  An operand is stored either with the reduction index contiguous ("KC":
// x, w in the forward pass, du in dx) or strided ("CM": w in dx, du and x in dw).  One tile kernel serves all of them: tiles of both
// operands are staged in LDS as 16-byte chunks, KC images are read as fragments of 8 consecutive reduction elements, CM images through
// the transposing LDS load (bf16) or element by element (fp32), and 32x32 MFMA tiles accumulate in fp32.  The MFMA computes the
// transposed tile (Q rows x P columns): a lane then holds 4 neighbouring output columns of one row.
#include "act8.h"
#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace {

template <class T> struct Frag;
template <> struct Frag<float> { float v[8]; };
template <> struct Frag<bf16_t> { bf16x8 v; };

// lane (r, h) holds reduction elements 8 h .. 8 h + 7 of its row; for fp32 the order inside the 16-deep step is a permutation applied
// to both operands
__device__ __forceinline__ void mma(f32x16& acc, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, const Frag<bf16_t>& a, const Frag<bf16_t>& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, acc, 0, 0, 0);
}

// Two transposing LDS loads, `second` bytes apart.  `restrict`: what it reads is not written while it runs, so that the compiler need not put a wait
// for every DMA under way before it; the kernel's own waits order the two.
__device__ __forceinline__ bf16x8 read_tr(const char* __restrict a, int second) {
    union { s16x4 s[2]; bf16x8 b; } c;
    c.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
    c.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + second));
    return c.b;
}

struct GemmP {
    const char *P, *Q;                    // operands
    long long ldp, ldq;                   // elements
    long long I, Cn;                      // output rows, reduction length
    int J;                                // output columns
    long long cchunk;                     // reduction elements of a split (a multiple of BK)
    int splits;
    int ti, tj;                           // tiles
    // output
    void* out; long long ldo;
    float* part;                          // splits > 1: [split][I][ldpart]
    int ldpart;                           // J rounded up to whole vectors of 8
    const float* bias;
    const void* res; long long ldr;
    void* pre; long long ldpre;
    int act;
};


// LDS image of one operand's tile (ROWS outputs x BKE reduction elements of T).
//   KC: [ROWS][BKE], rows of 128 bytes (8 chunks of 16); chunk ^= (row >> 1) & 7: any 16 consecutive rows read at one chunk index cover the
//       256 bytes of a bank row once.
//   CM bf16: [BKE][ROWS]; the transposing load reads, per half wave, one 64-byte piece of 4 consecutive rows: the piece index is XORed
//       with row & 3 so that the four lie in different quarters of the 256-byte bank row.
//   CM fp32: [BKE][ROWS]; the two halves of a wave read rows k and k + 8: the 128-byte half is XORed with bit 3 of the row.
template <class T, int ROWS, bool CM, int BKE_ = 128 / (int)sizeof(T)> struct TileImg {
    static constexpr int BKE = BKE_;
    static constexpr int RB = BKE * (int)sizeof(T);                   // bytes of a KC row: 64 or 128
    static constexpr int VE = 16 / sizeof(T);
    static constexpr int CPR = CM ? ROWS / VE : BKE / VE;             // chunks of a row
    static constexpr int CHUNKS = ROWS * BKE / VE;
    static constexpr int BYTES = CHUNKS * 16;
    static_assert(ROWS == 64 || ROWS == 128 || ROWS == 256, "swizzles");
    // (rows of 128 bytes put rows r and r + 2 on one quarter)
    __device__ static __forceinline__ int piece_swz(int row) { return ROWS == 64 ? (row >> 1) & 1 : row & 3; }
    __device__ static __forceinline__ int off(int row, int ch) {
        if constexpr (!CM) return row * RB + ((ch ^ ((row / (256 / RB)) & (CPR - 1))) << 4);
        else if constexpr (sizeof(T) == 2) return row * (ROWS * 2) + ((((ch >> 2) ^ piece_swz(row)) << 2 | (ch & 3)) << 4);
        else return row * (ROWS * 4) + ((ch ^ (row & 8)) << 4);
    }
    // inverse: which chunk of its row the 16-byte slot `slot` of that row holds
    __device__ static __forceinline__ int chunk_at(int row, int slot) { return (off(row, slot) - row * (CM ? ROWS * (int)sizeof(T) : RB)) >> 4; }
    // fragment: output row rb + (lane & 31), reduction elements k0 + 8 (lane >> 5) ..
    __device__ static __forceinline__ void frag(Frag<T>& f, const char* lds, int rb, int k0, int lane) {
        const int r = lane & 31, h = lane >> 5;
        if constexpr (!CM && sizeof(T) == 2) {
            f.v = *(const bf16x8*)(lds + off(rb + r, (k0 >> 3) + h));
        } else if constexpr (!CM) {
            const float4 lo = *(const float4*)(lds + off(rb + r, (k0 >> 2) + 2 * h)), hi = *(const float4*)(lds + off(rb + r, (k0 >> 2) + 2 * h + 1));
            f.v[0] = lo.x; f.v[1] = lo.y; f.v[2] = lo.z; f.v[3] = lo.w; f.v[4] = hi.x; f.v[5] = hi.y; f.v[6] = hi.z; f.v[7] = hi.w;
        } else if constexpr (sizeof(T) == 2) {
            const int i = lane & 15;
            const int row = k0 + 8 * h + (i >> 2);                    // and row + 4: the same swizzle
            const int ch = ((((rb >> 5) ^ piece_swz(row)) << 2) | (2 * ((lane >> 4) & 1) + ((i & 3) >> 1)));
            const char* a = lds + row * (ROWS * 2) + ch * 16 + 8 * (i & 1);
            f.v = read_tr(a, 4 * ROWS * 2);
        } else {
            const int ch = (rb + r) >> 2;
#pragma unroll
            for (int j = 0; j < 8; ++j) f.v[j] = *(const float*)(lds + off(k0 + 8 * h + j, ch) + 4 * (r & 3));
        }
    }
};

// 8 neighbouring elements of the residual, as they are in memory
template <class T> struct Raw8 { uint4 v[sizeof(T) / 2]; };
// FAST: all 8 exist, else `left` of them (zeros behind).  16-byte accesses at any alignment of the type: the memory system takes them, at a
// cost where they cross lines.
template <class T, bool FAST> __device__ __forceinline__ Raw8<T> load_res(const T* a, int left) {
    Raw8<T> r;
    if (FAST || left >= 8) __builtin_memcpy(&r, a, sizeof(r));
    else {
        float t[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = k < left ? to_f32<T>(a[k]) : 0.f;
        if constexpr (sizeof(T) == 2) vec_put(r.v[0], t);
        else __builtin_memcpy(&r, t, sizeof(r));
    }
    return r;
}
// 8 neighbouring output columns of a row, `left` of which exist: bias, activation, residual, store.  oo, op: element offsets in out and pre
template <class T, class OT, bool FAST> __device__ __forceinline__ void epilogue8(const GemmP& p, float (&f)[8], const float (&bias)[8], const Raw8<T>& res, int left, long long oo, long long op) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += bias[k];
    const auto put = [&](OT* o) __attribute__((always_inline)) {
        if (FAST || left >= 8) {
            if constexpr (sizeof(OT) == 2) { uint4 r; vec_put(r, f); __builtin_memcpy(o, &r, 16); }
            else { __builtin_memcpy(o, f, 16); __builtin_memcpy(o + 4, f + 4, 16); }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k < left) o[k] = from_f32<OT>(f[k]);
        }
    };
    if (p.pre) put((OT*)p.pre + op);
    with_act(p.act, [&](auto a) __attribute__((always_inline)) { act_apply<T, decltype(a)::value>(f); });
    if (p.res) {
        float t[8];
        if constexpr (sizeof(T) == 2) vec_get(t, res.v[0]);
        else __builtin_memcpy(t, &res, sizeof(t));
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] += t[k];
    }
    put((OT*)p.out + oo);
}
__device__ __forceinline__ void load_bias(const GemmP& p, float (&b)[8], int j) {
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = p.bias && j + k < p.J ? p.bias[j + k] : 0.f;
}

// Staging by DMA: 16-byte chunks go from memory into LDS without registers in between.  A wave's load instruction fills 64
// neighbouring 16-byte slots, so the swizzle is applied to the addresses: the lane that fills slot s of a row loads the chunk that
// belongs there.  The buffer descriptor's range check turns what lies outside the operand into zeros: lanes whose output row (or
// column) does not exist, or whose chunk lies past the end of the reduction, carry an offset with bit 31 set.
typedef __attribute__((address_space(3))) void* lds_ptr;
// B: bytes that a lane brings, 16, or 4 for fp32 operands of any alignment and width (a wave's load brings
// 256 bytes then: 4001 x 4003 x 4005 953 us, 4004 x 4004 x 4004 931; 777 x 201 x 523 8.3 us, 10.5 and a copy of 3 with 16 bytes).
template <class T, int ROWS, bool CM, int BKE, int NT, int B> struct Dma {
    typedef TileImg<T, ROWS, CM, BKE> Img;
    static constexpr int PER = 16 / B, VB = B / (int)sizeof(T), NC = Img::CHUNKS * PER / NT;      // lanes of a chunk, elements of a lane
    static_assert(Img::CHUNKS * PER % NT == 0 && (B == 16 || B == 4) && VB > 0, "whole chunks per thread");
    unsigned voff[NC];
    const char* base;                 // element (o0, first reduction element of this split), KC; (first, o0), CM
    long long step;                   // bytes between steps
    __device__ __forceinline__ void init(const char* p, long long ld, long long o0, long long no, long long c0) {
        base = p + ((CM ? c0 * ld + o0 : o0 * ld + c0) * (long long)sizeof(T));
        step = CM ? (long long)BKE * ld * (long long)sizeof(T) : (long long)Img::RB;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = ((int)threadIdx.x + i * NT) / PER, d = (int)threadIdx.x % PER, row = c / Img::CPR, e = Img::chunk_at(row, c - row * Img::CPR) * Img::VE + d * VB;
            const bool ok = CM ? o0 + e < no : o0 + row < no;
            voff[i] = ok ? (unsigned)row * (unsigned)(ld * (int)sizeof(T)) + (unsigned)e * (unsigned)sizeof(T) : 0x80000000u;
        }
    }
    // FULL: BKE reduction elements are left; otherwise `left` of them, the rest reads as zero
    template <bool FULL> __device__ __forceinline__ void issue(char* lds, int wave, int left) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            unsigned v = voff[i];
            if constexpr (!FULL) {
                const int c = ((int)threadIdx.x + i * NT) / PER, row = c / Img::CPR;
                v = (CM ? row : Img::chunk_at(row, c - row * Img::CPR) * Img::VE + (int)threadIdx.x % PER * VB) < left ? v : 0x80000000u;
            }
            if constexpr (B == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + (wave * 64 + i * NT) * 16), 16, (int)v, 0, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + (wave * 64 + i * NT) * 4), 4, (int)v, 0, 0, 0);
        }
        base += step;
    }
};

// block -> (split, tile): blocks are dealt to the 8 XCDs in turn; each XCD takes a contiguous run of tiles, bands of 8 tile rows walked
// column by column, so that the tiles running at one time share operand rows in one L2
__device__ __forceinline__ void gemm_tile(const GemmP& p, int& split, int& ti, int& tj) {
    const long long n = (long long)p.ti * p.tj * p.splits, per = n / 8, b = blockIdx.x;
    long long lb = b < per * 8 ? (b & 7) * per + (b >> 3) : b;
    split = (int)(lb / ((long long)p.ti * p.tj));
    lb -= (long long)split * p.ti * p.tj;
    const int band = (int)(lb / (8 * p.tj)), in_band = (int)(lb - (long long)band * 8 * p.tj), bh = min(8, p.ti - band * 8);
    tj = in_band / bh;
    ti = band * 8 + in_band - tj * bh;
}

// Output tile of a wave through LDS: 32 rows at a time in a region of its own, [32][NJ * 32 + 4] fp32, so that a lane ends up with 8
// neighbouring columns of a row, 16 bytes of bf16; its columns are the same in every row it takes.  The residual of the next 32 rows is on its
// way while 32 are written (65536 x 1024 x 1024 with gelu and residual: 178 us, 203 with a load at each use).
template <class T, class OT, int TI, int TJ, int WI, int WJ, int NI, int NJ, bool FAST>
__device__ __forceinline__ void epilogue_tiles(const GemmP& p, f32x16 (&acc)[NI][NJ], float* tile, long long i0, int j, int split, int lane, int wi) {
    constexpr int WC = NJ * 32, RS = WC + 4, LPR = WC / 8, EL = 32 * LPR / 64, STEP = 64 / LPR;
    const int r0 = lane / LPR, left = p.J - j;
    const long long i_lo = i0 + wi * (TI / WI) + r0;               // row of this lane; + 32 a + STEP e
    float bias[8];
    load_bias(p, bias, j);
    const bool with_res = p.res && p.splits == 1;
    Raw8<T> res[2][EL];
    const auto fetch = [&](Raw8<T> (&r)[EL], int a) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < EL; ++e) {
            const long long i = i_lo + 32 * a + STEP * e;
            r[e] = load_res<T, FAST>((const T*)p.res + i * p.ldr + j, FAST || i < p.I ? left : 0);
        }
    };
    if (with_res) fetch(res[0], 0);
    __syncthreads();
#pragma unroll
    for (int a = 0; a < NI; ++a) {
#pragma unroll
        for (int c = 0; c < NJ; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *(float4*)(tile + (lane & 31) * RS + c * 32 + 8 * e + 4 * (lane >> 5)) = make_float4(acc[a][c][4 * e], acc[a][c][4 * e + 1], acc[a][c][4 * e + 2], acc[a][c][4 * e + 3]);
        __builtin_amdgcn_wave_barrier();
        if (with_res && a + 1 < NI) fetch(res[(a + 1) & 1], a + 1);
        const float* src = tile + r0 * RS + (lane % LPR) * 8;
        const long long i = i_lo + 32 * a;
        long long oo = i * p.ldo + j, op = i * p.ldpre + j;
        if (p.splits > 1) {
            float* o = p.part + ((long long)split * p.I + i) * p.ldpart + j;
#pragma unroll FAST ? 4 : 1
            for (int e = 0; e < EL; ++e) {
                const float4 lo = *(const float4*)src, hi = *(const float4*)(src + 4);
                if (FAST || (i + e * STEP < p.I && left > 0)) { ((float4*)o)[0] = lo; ((float4*)o)[1] = hi; }
                src += STEP * RS;
                o += (long long)STEP * p.ldpart;
            }
        } else {
#pragma unroll
            for (int e = 0; e < EL; ++e) {
                const float4 lo = *(const float4*)src, hi = *(const float4*)(src + 4);
                float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                if (FAST || (i + e * STEP < p.I && left > 0)) {
                    epilogue8<T, OT, FAST>(p, f, bias, res[a & 1][e], left, oo, op);
                }
                src += STEP * RS;
                oo += STEP * p.ldo; op += STEP * p.ldpre;
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}
template <class T, class OT, int TI, int TJ, int WI, int WJ, int NI, int NJ>
__device__ __forceinline__ void gemm_epilogue(const GemmP& p, f32x16 (&acc)[NI][NJ], char* smem, long long i0, int j0, int split, int lane, int wi, int wj, int wave) {
    constexpr int WC = NJ * 32;
    float* tile = (float*)smem + wave * 32 * (WC + 4);
    const int j = j0 + wj * WC + (lane % (WC / 8)) * 8;
    if (i0 + TI <= p.I && j0 + TJ <= p.J) epilogue_tiles<T, OT, TI, TJ, WI, WJ, NI, NJ, true>(p, acc, tile, i0, j, split, lane, wi);
    else epilogue_tiles<T, OT, TI, TJ, WI, WJ, NI, NJ, false>(p, acc, tile, i0, j, split, lane, wi);
}

// Instruction order of a slice of M MFMAs with R LDS reads and `v` (0 or more) DMA loads: spread between the MFMAs
template <int M, int R> __device__ __forceinline__ void slice_order(const int v) {
#pragma unroll
    for (int i = 0; i < M; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        constexpr int per = (R + M - 1) / M;
        if (i * per < R) __builtin_amdgcn_sched_group_barrier(0x100, per, 0);
        if (i < v) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
}

// T: type of the operands and the residual, OT: of the output (and pre).  TI x TJ output tile, WI x WJ waves.
// Both operands are staged by DMA into a ring of STAGES tiles of BKE reduction elements.  A step has one barrier, before its last slice of 16:
// there every wave has the fragments of the rest of tile t in registers, so that its slot takes the DMA of tile t + STAGES, and tile t + 1 is
// waited for, whose first fragments are read beside the last slice's MFMAs.  So a load has STAGES - 1 steps to arrive, and no MFMA waits for LDS
// behind a barrier.  Bound by the matrix units and, close behind, LDS (a wave's 128 x 64 tile reads 6 fragments for 8 MFMAs): 16384 x 4096 x 4096
// bf16 418 to 430 us, 1280 to 1315 TFLOP/s; 4096 x 4096 x 4096 fp32 940 us, 146.
// (fp32 with a row operand: the two 16-byte LDS loads of a fragment are no builtins with `restrict`, and the compiler waits for every DMA under way
// before them, so that a load has part of a step to arrive.)
template <class T, class OT, int TI, int TJ, int WI, int WJ, int BKE, int STAGES, bool PCM, bool QCM, int WPE, int B>
__global__ __launch_bounds__(64 * WI * WJ, WPE) void gemm_dma_kernel(const GemmP p) {
    constexpr int NT = 64 * WI * WJ;
    typedef TileImg<T, TI, PCM, BKE> PI;
    typedef TileImg<T, TJ, QCM, BKE> QI;
    constexpr int STAGE = PI::BYTES + QI::BYTES, SL = BKE / 16;
    constexpr int NI = TI / WI / 32, NJ = TJ / WJ / 32;
    constexpr int LOADS = Dma<T, TI, PCM, BKE, NT, B>::NC + Dma<T, TJ, QCM, BKE, NT, B>::NC;   // DMA instructions of a wave per step
    static_assert(STAGES >= 2 && SL >= 2 && SL % 2 == 0, "ring and slices");
    extern __shared__ char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wi = wave / WJ, wj = wave - wi * WJ;
    int split, ti, tj;
    gemm_tile(p, split, ti, tj);
    const long long i0 = (long long)ti * TI;
    const int j0 = tj * TJ;
    const long long cb = split * p.cchunk, ce = min(p.Cn, cb + p.cchunk);

    f32x16 acc[NI][NJ];
#pragma unroll
    for (int a = 0; a < NI; ++a)
#pragma unroll
        for (int c = 0; c < NJ; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][c][e] = 0.f;

    Dma<T, TI, PCM, BKE, NT, B> dp;
    Dma<T, TJ, QCM, BKE, NT, B> dq;
    dp.init(p.P, p.ldp, i0, p.I, cb);
    dq.init(p.Q, p.ldq, j0, p.J, cb);
    const int steps = (int)((ce - cb + BKE - 1) / BKE);
    const int pb = wi * (TI / WI), qb = wj * (TJ / WJ);
    const int last = (int)(ce - cb - (long long)(steps - 1) * BKE);       // reduction elements of the last step
    const auto issue = [&](char* s, int t) __attribute__((always_inline)) {
        if (t + 1 < steps) {
            dp.template issue<true>(s, wave, BKE);
            dq.template issue<true>(s + PI::BYTES, wave, BKE);
        } else {
            dp.template issue<false>(s, wave, last);
            dq.template issue<false>(s + PI::BYTES, wave, last);
        }
    };
    if (steps > 0) {
        for (int t = 0; t < STAGES && t < steps; ++t) issue(smem + t * STAGE, t);
        // tile 0 has landed
        if (steps >= STAGES) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
        Frag<T> fp[2][NI], fq[2][NJ];
#pragma unroll
        for (int a = 0; a < NI; ++a) PI::frag(fp[0][a], smem, pb + a * 32, 0, lane);
#pragma unroll
        for (int c = 0; c < NJ; ++c) QI::frag(fq[0][c], smem + PI::BYTES, qb + c * 32, 0, lane);
        char* cur = smem;
        // FULL: another whole tile to load
        const auto step = [&](int t, auto full) __attribute__((always_inline)) {
            constexpr bool FULL = decltype(full)::value;
            char* nxt = cur + STAGE == smem + STAGES * STAGE ? smem : cur + STAGE;
#pragma unroll
            for (int k = 0; k < SL; ++k) {
                __builtin_amdgcn_sched_barrier(0);
                if (k + 1 == SL) {
                    // this wave's reads of tile t are done and its part of tile t + 1 has landed (younger loads may be under way)
                    if (FULL || t + STAGES <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * LOADS) : "memory");
                    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    asm volatile("s_barrier" ::: "memory");
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (FULL) {
                        dp.template issue<true>(cur, wave, BKE);
                        dq.template issue<true>(cur + PI::BYTES, wave, BKE);
                    } else if (t + STAGES < steps) issue(cur, t + STAGES);
                }
                const char* s = k + 1 < SL ? cur : nxt;
                const int k1 = k + 1 < SL ? (k + 1) * 16 : 0;
                // (past the last tile this reads a slot that holds older values, and nothing uses them)
#pragma unroll
                for (int c = 0; c < NJ; ++c) QI::frag(fq[(k + 1) & 1][c], s + PI::BYTES, qb + c * 32, k1, lane);
#pragma unroll
                for (int a = 0; a < NI; ++a) PI::frag(fp[(k + 1) & 1][a], s, pb + a * 32, k1, lane);
#pragma unroll
                for (int a = 0; a < NI; ++a)
#pragma unroll
                    for (int c = 0; c < NJ; ++c) mma(acc[a][c], fq[k & 1][c], fp[k & 1][a]);
                // order of the slice: an MFMA, then a share of the LDS reads and (last slice) of the DMA instructions, and so on
                if constexpr (sizeof(T) == 2) slice_order<NI * NJ, (PCM ? 2 : 1) * NI + (QCM ? 2 : 1) * NJ>(k + 1 == SL && FULL ? LOADS : 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            cur = nxt;
        };
        int t = 0;
        for (; t + STAGES + 1 < steps; ++t) step(t, std::true_type());
        for (; t < steps; ++t) step(t, std::false_type());
    }
    gemm_epilogue<T, OT, TI, TJ, WI, WJ>(p, acc, smem, i0, j0, split, lane, wi, wj, wave);
}

// Sum of the splits, then the epilogue
template <class T, class OT> __global__ __launch_bounds__(256) void gemm_join_kernel(const GemmP p) {
    const int per_row = p.ldpart / 8;
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long i = t / per_row;
    const int j = (int)(t - i * per_row) * 8;
    if (i >= p.I) return;
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.f;
    const float* a = p.part + i * p.ldpart + j;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float4 lo = ((const float4*)a)[0], hi = ((const float4*)a)[1];
        f[0] += lo.x; f[1] += lo.y; f[2] += lo.z; f[3] += lo.w; f[4] += hi.x; f[5] += hi.y; f[6] += hi.z; f[7] += hi.w;
        a += p.I * p.ldpart;
    }
    float bias[8];
    load_bias(p, bias, j);
    Raw8<T> res;
    if (p.res) res = load_res<T, false>((const T*)p.res + i * p.ldr + j, p.J - j);
    epilogue8<T, OT, false>(p, f, bias, res, p.J - j, i * p.ldo + j, i * p.ldpre + j);
}

// ---- few rows --------------------------------------------------------------------------------------------------------------
// x w^T for M up to 16 rows (one to a few samples): bound by reading w once, so nothing is staged.  A block takes 16 columns (rows of w)
// and all of K: its 16 waves take 32-deep (fp32: 16-deep) slices in turn and feed 16-byte loads straight into 16x16 MFMA; the waves' sums
// meet in LDS.  Rows of x or w that do not exist repeat the last one and are not stored.  1 x 4096 x 4096 bf16: 8.2 us, 4.1 TB/s of w; the
// tile kernels take 15.  (For 32 and 64 rows of 4096 x 4096, with 2 and 4 row tiles of x a wave, 14 and 22 us against their 15 and 16: not kept.)
typedef float f32x4_t __attribute__((ext_vector_type(4)));
template <class T> __device__ __forceinline__ uint4 load_chunk(const T* row, int k, int K) { return load16(row + k, K - k); }     // from element k; past K zeros
template <class T> __device__ __forceinline__ void mma16(f32x4_t& acc, const uint4& a, const uint4& b) {
    if constexpr (sizeof(T) == 2) {
        union { uint4 u; bf16x8 v; } x, y;
        x.u = a; y.u = b;
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, y.v, acc, 0, 0, 0);
    } else {
        const unsigned ax[4] = {a.x, a.y, a.z, a.w}, bx[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ax[j]), __uint_as_float(bx[j]), acc, 0, 0, 0);
    }
}
constexpr int SKINNY_M = 16;
template <class T> __global__ __launch_bounds__(1024) void skinny_kernel(const GemmP p) {
    constexpr int VE = 16 / sizeof(T), DEPTH = 4 * VE, AHEAD = 4;      // reduction elements of a slice; slices loaded together
    __shared__ float red[16][256 + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kq = lane >> 4;
    const int j0 = blockIdx.x * 16, K = (int)p.Cn;
    const T* w = (const T*)p.Q + (long long)min(j0 + r, p.J - 1) * p.ldq;
    const T* x = (const T*)p.P + min((long long)r, p.I - 1) * p.ldp;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = wave * DEPTH; k0 < K; k0 += 16 * DEPTH * AHEAD) {
        uint4 a[AHEAD], b[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int k = k0 + u * 16 * DEPTH + kq * VE;
            a[u] = load_chunk(w, k, K);
            b[u] = load_chunk(x, k, K);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) mma16<T>(acc, a[u], b[u]);
    }
    *(float4*)&red[wave][r * 16 + 4 * kq] = make_float4(acc[0], acc[1], acc[2], acc[3]);   // [row of x][column]
    __syncthreads();
    if (threadIdx.x < 256) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) s += red[v][threadIdx.x];
        red[0][threadIdx.x] = s;                           // (each thread its own column of red)
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int i = threadIdx.x >> 1, c = (threadIdx.x & 1) * 8, j = j0 + c;
        if (i < p.I && j < p.J) {
            float f[8], bias[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = red[0][i * 16 + c + k];
            load_bias(p, bias, j);
            Raw8<T> res;
            if (p.res) res = load_res<T, false>((const T*)p.res + i * p.ldr + j, p.J - j);
            epilogue8<T, T, false>(p, f, bias, res, p.J - j, i * p.ldo + j, i * p.ldpre + j);
        }
    }
}

// ---- operands for DMA ----------------------------------------------------------------------------------------------------
// Copy of up to three operands [rows][cols] with any stride and alignment into [rows][ldo], ldo a multiple of 16 bytes, the rest of a row
// zero: bf16 rows that are not 16-byte aligned, and rows more than 4 MB apart.  One pass over an odd operand costs less than staging it through
// registers would in every tile (x w^T 777 x 201 x 523 bf16: 14 us against 10).
struct PackP { const char* src[3]; long long ld[3]; char* dst[3]; long long rows[3], first[4]; int cols[3], cpr[3]; };   // cpr: 16-byte chunks of an output row; first: blocks
template <class T> __global__ __launch_bounds__(256) void pack_kernel(const PackP p) {
    const int j = (blockIdx.x >= p.first[1]) + (blockIdx.x >= p.first[2]);
    const long long t = ((long long)blockIdx.x - p.first[j]) * 256 + threadIdx.x;
    const long long row = t / p.cpr[j];
    const int ch = (int)(t - row * p.cpr[j]);
    if (row < p.rows[j]) ((uint4*)p.dst[j])[t] = load_chunk((const T*)p.src[j] + row * p.ld[j], ch * (16 / (int)sizeof(T)), p.cols[j]);
}

// ---- du = dy act'(u) and the column sums of du ---------------------------------------------------------------------------
// A block takes 64 vectors of columns of a run of rows, 4 rows at a time; column sums (fp32) of the unrounded du go to part[run][N].  du is
// rounded to T, since the matrix units read operands of that type, and written with rows of ldu elements, zero past N.  For bf16 that makes the error
// of dx and dw 0.0023 of their norm, 0.0017 with an unrounded du (the rounding of the result), at 65536 x 1024 x 1024; a du of two bf16 parts would
// take both products twice, 270 us more.  Against the formula with du rounded once, 0.03 to 0.2 % of the values are one step off.  Bound by memory: 65536 x 1024 bf16 gelu
// 81 to 88 us, 4.6 to 5.0 TB/s; 16384 x 4096 from a checkpoint 67 to 69 us.
struct DuP {
    const void* dy; long long lddy;
    const void* pre; long long ldpre;
    const unsigned char *pq, *pe; long long ldpe;
    void* du; long long ldu;               // NULL: sums only
    float* part;                           // NULL: no sums
    long long M, rows;
    int N, act;
};
template <class T, int SRC> __global__ __launch_bounds__(256) void act_bwd_kernel(const DuP p) {   // SRC: 0 no activation, 1 pre, 2 checkpoint
    constexpr int V = 16 / sizeof(T);
    __shared__ float red[4][64 * V];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int j = blockIdx.x * (64 * V) + lane * V;
    const long long r0 = (long long)blockIdx.y * p.rows, r1 = min(p.M, r0 + p.rows);
    float s[V];
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = 0.f;
    if (j < p.N)
        with_act(SRC == 0 ? FAVAE_ACT_NONE : p.act, [&](auto a) __attribute__((always_inline)) {
#pragma unroll 4
            for (long long i = r0 + w; i < r1; i += 4) {
                uint4 rd = load_chunk((const T*)p.dy + i * p.lddy, j, p.N);
                float d[V];
                vec_get(d, rd);
                if constexpr (SRC > 0) {
                    float z[V];
                    if constexpr (SRC == 1) {
                        vec_get(z, load_chunk((const T*)p.pre + i * p.ldpre, j, p.N));
                    } else {
                        const float sc = ck_scale(p.pe[i * p.ldpe + (j >> 5)]);
                        const unsigned char* a8 = p.pq + i * p.ldpre + j;
                        unsigned wd[2] = {0u, 0u};
                        if (j + V <= p.N) __builtin_memcpy(wd, a8, V);
                        else
#pragma unroll
                            for (int k = 0; k < V; ++k) if (j + k < p.N) wd[k >> 2] |= (unsigned)a8[k] << (8 * (k & 3));
#pragma unroll
                        for (int k = 0; k < V; ++k) z[k] = ck_value(wd[k >> 2], k & 3, sc);
                    }
                    act_grad_mul<T, decltype(a)::value>(d, z);       // (past N: dy is 0, and z is 0 or, in a faulty block, NaN)
#pragma unroll
                    for (int k = 0; k < V; ++k) d[k] = j + k < p.N ? d[k] : 0.f;
                    vec_put(rd, d);
                }
                if (p.du) *(uint4*)((T*)p.du + i * p.ldu + j) = rd;
#pragma unroll
                for (int k = 0; k < V; ++k) s[k] += d[k];
            }
        });
    if (!p.part) return;
#pragma unroll
    for (int k = 0; k < V; ++k) red[w][lane * V + k] = s[k];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * V; k += 256) {
        const int c = blockIdx.x * (64 * V) + k;
        if (c < p.N) p.part[(long long)blockIdx.y * p.N + c] = (red[0][k] + red[1][k]) + (red[2][k] + red[3][k]);
    }
}
__global__ __launch_bounds__(512) void col_join_kernel(const float* __restrict__ part, long long rows, int N, float* __restrict__ out) {
    __shared__ float red[32][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4;
    float s = 0.f;
    if (c < N)
#pragma unroll 4
        for (long long i = k; i < rows; i += 32) s += part[i * N + c];
    red[k][threadIdx.x & 15] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < N) {
        float t = 0.f;
        for (int i = 0; i < 32; ++i) t += red[i][threadIdx.x];
        out[c] = t;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------
bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

constexpr long long CUS = 256;
// Tiles of the product kernels: WIDE (bf16) where a CU has the one workgroup that its LDS takes, SMALL and TINY where tiles are few.
// A reduction may be split over workgroups, whose fp32 sums a second launch joins.  Tile and splits are those with the least estimated
// time, from what a step (128 bytes of reduction) was measured to take (us): alone on its CU, and as a share of a full one.
//   bf16   WIDE 1.55 / 1.55   SMALL 0.66 / 0.63   TINY 0.33 / 0.2
//   fp32                      SMALL 1.95 / 1.83   TINY 0.72 / 0.48
// Both sides (us): x w^T, du w of 2048 x 2048 x 2048 bf16 SMALL 22, 22, TINY 28, 30; of 1024 x 1024 x 1024 11, 11 and 7.2, 7.3; of 2048 x 2048 x
// 2048 fp32 128, 131 and 141, 146; of 1024 x 1024 x 1024 63, 65 and 23, 25.
enum Tile { WIDE = 0, SMALL = 1, TINY = 2 };
constexpr int TILE_I[3] = {256, 128, 64}, TILE_PER_CU[3] = {1, 2, 4};      // square; workgroups that share a CU
struct GemmPlan { Tile tile; int splits; };
GemmPlan plan_gemm(long long I, int J, long long Cn, int es) {
    constexpr double ALONE[2][3] = {{1.55, 0.66, 0.33}, {0, 1.95, 0.72}}, SHARE[2][3] = {{1.55, 0.63, 0.2}, {0, 1.83, 0.48}};
    const long long steps = std::max<long long>(1, cdivll(Cn * es, 128));
    GemmPlan best = {TINY, 1};
    double least = 1e30;
    for (int t = es == 2 ? WIDE : SMALL; t <= TINY; ++t) {
        const double alone = ALONE[es == 4][t], share = SHARE[es == 4][t];
        const long long tiles = cdivll(I, TILE_I[t]) * cdivll(J, TILE_I[t]);
        const double epilogue = TILE_I[t] * TILE_I[t] * 1.2e-4;                     // 2 us for 128 x 128
        for (int s = 1; s <= 64; s += s < 4 ? 1 : s < 16 ? 4 : 16) {
            if (s > 1 && (steps < 2 * s || tiles * s > 4096)) break;
            const long long per_cu = cdivll(tiles * s, CUS), rounds = cdivll(per_cu, TILE_PER_CU[t]);
            const double beside = (double)std::min<long long>(per_cu, TILE_PER_CU[t]);
            const double us = rounds * (cdivll(steps, s) * std::max(alone, beside * share) + 1.5 + beside * epilogue) +
                              (s > 1 ? 4.0 + s * (double)I * J * 2e-6 : 0.0);
            if (us < least) { least = us; best = {(Tile)t, s}; }
        }
    }
    return best;
}

template <class T, class OT, int TI, int TJ, int WI, int WJ, int BKE, int STAGES, bool PCM, bool QCM, int WPE, int B = 16>
void gemm_launch(const GemmP& p, unsigned blocks, hipStream_t st) {
    constexpr size_t ring = STAGES * (size_t)(TileImg<T, TI, PCM, BKE>::BYTES + TileImg<T, TJ, QCM, BKE>::BYTES);
    constexpr size_t lds = std::max(ring, (size_t)WI * WJ * 32 * (TJ / WJ + 4) * sizeof(float));
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    gemm_dma_kernel<T, OT, TI, TJ, WI, WJ, BKE, STAGES, PCM, QCM, WPE, B><<<blocks, 64 * WI * WJ, lds, st>>>(p);
}

// out = P Q^T over operands that DMA can take: 16-byte aligned rows, a whole number of chunks (the rest of a KC row zero), and 32-bit offsets
// inside a tile; odd (fp32): any alignment and width
template <class T, class OT, bool PCM, bool QCM> int gemm_run(GemmP p, bool odd, hipStream_t st) {
    if (p.I == 0 || p.J == 0) return FAVAE_OK;
    constexpr int es = sizeof(T);
    const GemmPlan pl = plan_gemm(p.I, p.J, p.Cn, es);
    p.ti = (int)cdivll(p.I, TILE_I[pl.tile]);
    p.tj = cdiv(p.J, TILE_I[pl.tile]);
    const long long unit = 128 / es;
    p.cchunk = cdivll(cdivll(p.Cn, unit), pl.splits) * unit;
    p.splits = (int)std::max<long long>(1, cdivll(p.Cn, std::max<long long>(1, p.cchunk)));
    const unsigned blocks = (unsigned)p.ti * (unsigned)p.tj * (unsigned)p.splits;
    p.ldpart = (p.J + 7) & ~7;
    // steps of 128 bytes and two stages; one 64-byte steps and four where neither operand's steps leave half lines behind (x w^T 16384 x 4096 x
    // 4096: 430 us, 452 with 64-byte steps; du w 423, 434; du^T x 409, 406; with 1024 rows and columns over 65536: 136, 131) and in SMALL, for
    // loads that are longer under way (2048 x 2048 x 2048: 22.3 us, 26).  TINY with a CU to itself: four stages, where two leave too little of w
    // under way (64 x 4096 x 4096 13 us, 15.5; fp32 33 either way, for the wait named at gemm_dma_kernel); with neighbours 30 us, 34 (du w 2048 x 2048 x 2048) the other way round.
    if constexpr (es == 4) {
        if (pl.tile == TINY && odd) gemm_launch<T, OT, 64, 64, 2, 2, 32, 2, PCM, QCM, 2, 4>(p, blocks, st);
        else if (pl.tile == TINY) gemm_launch<T, OT, 64, 64, 2, 2, 32, 2, PCM, QCM, 2>(p, blocks, st);
        else if (odd) gemm_launch<T, OT, 128, 128, 2, 4, 32, 2, PCM, QCM, 4, 4>(p, blocks, st);
        else gemm_launch<T, OT, 128, 128, 2, 4, 32, 2, PCM, QCM, 4>(p, blocks, st);
    } else if (pl.tile == TINY && blocks <= CUS) gemm_launch<T, OT, 64, 64, 2, 2, 64, 4, PCM, QCM, 2>(p, blocks, st);
    else if (pl.tile == TINY) gemm_launch<T, OT, 64, 64, 2, 2, 64, 2, PCM, QCM, 2>(p, blocks, st);
    else if (pl.tile == SMALL) gemm_launch<T, OT, 128, 128, 2, 2, 32, 4, PCM, QCM, 2>(p, blocks, st);
    else if constexpr (PCM && QCM) gemm_launch<T, OT, 256, 256, 2, 4, 32, 4, PCM, QCM, 2>(p, blocks, st);
    else gemm_launch<T, OT, 256, 256, 2, 4, 64, 2, PCM, QCM, 2>(p, blocks, st);
    FAVAE_LAUNCH_CHECK();
    if (p.splits > 1) {
        gemm_join_kernel<T, OT><<<(unsigned)cdivll(p.I * (p.ldpart / 8), 256), 256, 0, st>>>(p);
        FAVAE_LAUNCH_CHECK();
    }
    return FAVAE_OK;
}

// Operands as DMA takes them, or copies of them in the workspace (`ours`: rows padded to 16 bytes).  odd: 1 if a row is not 16-byte aligned, 2 if
// rows are more than 4 MB apart.
struct Operand { const char* p; long long ld, rows; int cols; bool ours = false; };
int odd_of(const Operand& o, int es) { return o.ld * es > 1 << 22 ? 2 : !aligned(o.p, 16) || (o.ld * es) % 16 != 0; }
bool dma16(const Operand& o, int es) { return o.ours || (odd_of(o, es) == 0 && (o.cols * es) % 16 == 0); }
bool dma_ok(const Operand& o, int es) { return dma16(o, es) || (es == 4 && odd_of(o, es) < 2); }
long long padded(long long cols, int es) { return cdivll(cols * es, 16) * 16 / es; }
size_t pack_bytes(long long rows, int cols, int es);
template <class T> int pack_operands(std::initializer_list<Operand*> ops, char*& ws, hipStream_t st) {
    PackP k = {};
    int n = 0;
    for (Operand* o : ops) {
        if (!o || o->rows == 0 || o->cols == 0 || dma_ok(*o, sizeof(T))) continue;
        const long long ldo = padded(o->cols, sizeof(T));
        k.src[n] = o->p; k.ld[n] = o->ld; k.dst[n] = ws; k.rows[n] = o->rows; k.cols[n] = o->cols; k.cpr[n] = (int)(ldo * (int)sizeof(T) / 16);
        k.first[n + 1] = k.first[n] + cdivll(o->rows * k.cpr[n], 256);
        *o = {ws, ldo, o->rows, o->cols, true};
        ws += pack_bytes(o->rows, o->cols, sizeof(T));
        ++n;
    }
    if (n == 0) return FAVAE_OK;
    for (int j = n + 1; j < 4; ++j) k.first[j] = k.first[n];
    pack_kernel<T><<<(unsigned)k.first[n], 256, 0, st>>>(k);
    FAVAE_LAUNCH_CHECK();
    return FAVAE_OK;
}

size_t round256(size_t a) { return (a + 255) & ~(size_t)255; }
size_t pack_bytes(long long rows, int cols, int es) { return round256((size_t)rows * padded(cols, es) * es); }
size_t split_bytes(long long I, int J, long long Cn, int es) {
    if (I == 0 || J == 0) return 0;
    const int s = plan_gemm(I, J, Cn, es).splits;
    return s > 1 ? round256((size_t)s * I * ((J + 7) & ~7) * sizeof(float)) : 0;
}
constexpr int DU_RUNS = 256;
// rows of a run; up to 64 rows are one run, whose sums are db: no launch to join them
long long du_rows(long long M) { return M <= 64 ? 64 : std::max<long long>(16, cdivll(M, DU_RUNS)); }

int lin_sizes(const char* who, long long M, int N, int K, int act, int dtype) {
    FAVAE_CHECK_ARG(dtype == FAVAE_F32 || dtype == FAVAE_BF16, "%s: dtype is neither fp32 nor bf16", who);
    FAVAE_CHECK_ARG(act >= FAVAE_ACT_NONE && act <= FAVAE_ACT_GELU_TANH, "%s: unknown activation %d", who, act);
    FAVAE_CHECK_ARG(M >= 0 && N >= 0 && K >= 0 && M <= 0x7fffffffLL && N <= (1 << 20) && K <= (1 << 20), "%s: a size is negative or too large", who);
    // 512 GB of bf16: no tensor of the card, and every launch below stays under 2^31 workgroups (operands copied 256 chunks of 16 bytes at a time: two of
    // 2^38 fp32 and a w of 2^40 are 1.5 * 2^30; tiles of 64 x 64: 2^28)
    FAVAE_CHECK_ARG(M * std::max(N, K) <= 1LL << 38, "%s: %lld rows of %d and %d columns are too large", who, M, N, K);
    return FAVAE_OK;
}

// Whether operands [..][cols] need no copy, from their width and the largest of their `odd`
bool whole(int cols, int es, int odd) { return es == 4 ? odd < 2 : !odd && (cols * es) % 16 == 0; }

struct FwdScratch { size_t split, total; };
FwdScratch fwd_scratch(long long M, int N, int K, int odd, int es) {
    if (M == 0 || N == 0 || M <= SKINNY_M) return {0, 0};
    FwdScratch s;
    s.split = split_bytes(M, N, K, es);
    s.total = s.split + (whole(K, es, odd) ? 0 : pack_bytes(M, K, es) + pack_bytes(N, K, es));
    return s;
}
template <class T> int lin_fwd(GemmP p, Operand x, Operand w, char* scratch, const FwdScratch& sz, hipStream_t st) {
    p.part = (float*)scratch;
    if (x.rows <= SKINNY_M) {
        p.P = x.p; p.ldp = x.ld; p.Q = w.p; p.ldq = w.ld;
        p.splits = 1;
        skinny_kernel<T><<<(unsigned)cdiv(p.J, 16), 1024, 0, st>>>(p);
        FAVAE_LAUNCH_CHECK();
        return FAVAE_OK;
    }
    char* ws = scratch + sz.split;
    const int rc = pack_operands<T>({&x, &w}, ws, st);
    if (rc != FAVAE_OK) return rc;
    p.P = x.p; p.ldp = x.ld; p.Q = w.p; p.ldq = w.ld;
    return gemm_run<T, T, false, false>(p, !(dma16(x, sizeof(T)) && dma16(w, sizeof(T))), st);
}

struct BwdScratch { size_t du, colp, split, total; long long ldu; bool need_du; };
BwdScratch bwd_scratch(long long M, int N, int K, int act, bool x_ckpt, int odd, int es) {
    BwdScratch s;
    s.ldu = padded(N, es);
    s.need_du = act != FAVAE_ACT_NONE || !whole(N, es, odd);      // du, or dy as DMA takes it (then in either of two places)
    s.du = s.need_du ? pack_bytes(M, N, es) : 0;
    s.colp = M > 0 ? round256((size_t)cdivll(M, du_rows(M)) * N * sizeof(float)) : 0;
    s.split = std::max(split_bytes(M, K, N, es), split_bytes(N, K, M, es));    // the two products run one after the other
    s.total = s.du + s.colp + s.split + (act == FAVAE_ACT_NONE ? s.du : 0) + (whole(K, es, odd) ? 0 : pack_bytes(N, K, es)) + (whole(K, es, odd) && !x_ckpt ? 0 : pack_bytes(M, K, es));
    return s;
}

template <class T> int lin_bwd(Operand dy, Operand x, const unsigned char* xe, long long ldxe, Operand w, const void* pre, long long ldpre,
                               const unsigned char* pe, long long ldpe, long long M, int N, int K, int act, void* dx, long long lddx, void* dw,
                               long long lddw, int dw_f32, float* db, char* scratch, const BwdScratch& sz, hipStream_t st) {
    constexpr int es = sizeof(T);
    float* colp = (float*)(scratch + sz.du);
    float* part = (float*)(scratch + sz.du + sz.colp);
    char* ws = scratch + sz.du + sz.colp + sz.split;
    // du, or (beside the column sums) dy as DMA takes it
    const bool want_du = (dx || dw) && (act != FAVAE_ACT_NONE || (db && !dma_ok(dy, es)));
    const bool one_run = M > 0 && M <= du_rows(M);
    if (M > 0 && N > 0 && (want_du || db)) {
        DuP d = {dy.p, dy.ld, pre, ldpre, (const unsigned char*)pre, pe, ldpe, want_du ? scratch : nullptr, sz.ldu, db ? (one_run ? db : colp) : nullptr, M, du_rows(M), N, act};
        const dim3 g((unsigned)cdiv(N, 64 * (16 / es)), (unsigned)cdivll(M, d.rows));
        if (act == FAVAE_ACT_NONE) act_bwd_kernel<T, 0><<<g, 256, 0, st>>>(d);
        else if (!pe) act_bwd_kernel<T, 1><<<g, 256, 0, st>>>(d);
        else act_bwd_kernel<T, 2><<<g, 256, 0, st>>>(d);
        FAVAE_LAUNCH_CHECK();
        if (want_du) dy = {scratch, sz.ldu, M, N, true};
    }
    if (db && N > 0 && !one_run) {
        col_join_kernel<<<cdiv(N, 16), 512, 0, st>>>(colp, M > 0 ? cdivll(M, du_rows(M)) : 0, N, db);
        FAVAE_LAUNCH_CHECK();
    }
    if (dw && xe && M > 0 && K > 0) {
        // a checkpoint is decoded into the workspace first: 2 + 1 bytes a value, against decoding in the product's staging, which
        // made du^T x 283 us instead of 12 + 135 (4096 x 1024 x 16384)
        const long long ldt = padded(K, es);
        const int rc = favae_ckpt8_unpack(x.p, x.ld, xe, ldxe, M, K, ws, ldt, es == 4 ? FAVAE_F32 : FAVAE_BF16, st);
        if (rc != FAVAE_OK) return rc;
        x = {ws, ldt, M, K, true};
        ws += pack_bytes(M, K, es);
    }
    const int rc = pack_operands<T>({(dx || dw) && !want_du ? &dy : nullptr, dw && !xe ? &x : nullptr, dx ? &w : nullptr}, ws, st);
    if (rc != FAVAE_OK) return rc;
    GemmP p = {};
    p.P = dy.p; p.ldp = dy.ld; p.part = part; p.act = FAVAE_ACT_NONE;
    if (dx) {
        p.Q = w.p; p.ldq = w.ld; p.I = M; p.J = K; p.Cn = N; p.out = dx; p.ldo = lddx;
        const int r2 = gemm_run<T, T, false, true>(p, !(dma16(dy, es) && dma16(w, es)), st);
        if (r2 != FAVAE_OK) return r2;
    }
    if (dw) {
        p.Q = x.p; p.ldq = x.ld; p.I = N; p.J = K; p.Cn = M; p.out = dw; p.ldo = lddw;
        const bool odd = !(dma16(dy, es) && dma16(x, es));
        if constexpr (es == 2) {
            if (dw_f32) return gemm_run<T, float, true, true>(p, odd, st);
        }
        return gemm_run<T, T, true, true>(p, odd, st);
    }
    return FAVAE_OK;
}

}  // namespace

extern "C" size_t favae_linear_act_fwd_scratch(long long M, int N, int K, int odd, int dtype) {
    if (lin_sizes("favae_linear_act_fwd_scratch", M, N, K, FAVAE_ACT_NONE, dtype) != FAVAE_OK) return 0;
    return fwd_scratch(M, N, K, odd, dtype == FAVAE_F32 ? 4 : 2).total;
}

extern "C" int favae_linear_act_fwd(const void* x, long long ldx, const void* w, long long ldw, const float* bias, const void* residual,
                                    long long ldr, void* pre, long long ldpre, void* y, long long ldy, long long M, int N, int K, int act,
                                    void* scratch, size_t scratch_bytes, int dtype, void* stream) {
    const int rc = lin_sizes("favae_linear_act_fwd", M, N, K, act, dtype);
    if (rc != FAVAE_OK) return rc;
    if (M == 0 || N == 0) return FAVAE_OK;
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(y && (K == 0 || (x && w)), "favae_linear_act_fwd: null pointer");
    FAVAE_CHECK_ARG(ldy >= N && ldx >= K && ldw >= K && (!residual || ldr >= N) && (!pre || ldpre >= N), "favae_linear_act_fwd: a row stride is below the row's length");
    FAVAE_CHECK_ARG(aligned(x, es) && aligned(w, es) && aligned(y, es) && aligned(residual, es) && aligned(pre, es), "favae_linear_act_fwd: a pointer is not aligned to its type");
    const Operand ox = {(const char*)x, ldx, M, K}, ow = {(const char*)w, ldw, N, K};
    const FwdScratch sz = fwd_scratch(M, N, K, std::max(odd_of(ox, es), odd_of(ow, es)), es);
    FAVAE_CHECK_ARG(sz.total <= scratch_bytes && (sz.total == 0 || scratch) && aligned(scratch, 16), "favae_linear_act_fwd: scratch of %zu bytes, %zu needed", scratch_bytes, sz.total);
    GemmP p = {};
    p.I = M; p.J = N; p.Cn = K;
    p.out = y; p.ldo = ldy; p.bias = bias; p.res = residual; p.ldr = ldr; p.pre = pre; p.ldpre = ldpre; p.act = act;
    return dtype == FAVAE_F32 ? lin_fwd<float>(p, ox, ow, (char*)scratch, sz, (hipStream_t)stream)
                              : lin_fwd<bf16_t>(p, ox, ow, (char*)scratch, sz, (hipStream_t)stream);
}

extern "C" size_t favae_linear_act_bwd_scratch(long long M, int N, int K, int act, int x_ckpt, int odd, int dtype) {
    if (lin_sizes("favae_linear_act_bwd_scratch", M, N, K, act, dtype) != FAVAE_OK) return 0;
    return bwd_scratch(M, N, K, act, x_ckpt != 0, odd, dtype == FAVAE_F32 ? 4 : 2).total;
}

extern "C" int favae_linear_act_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* xe, long long ldxe, const void* w,
                                    long long ldw, const void* pre, long long ldpre, const void* pe, long long ldpe, long long M, int N, int K,
                                    int act, void* dx, long long lddx, void* dw, long long lddw, int dw_dtype, float* db, void* scratch,
                                    size_t scratch_bytes, int dtype, void* stream) {
    const int rc = lin_sizes("favae_linear_act_bwd", M, N, K, act, dtype);
    if (rc != FAVAE_OK) return rc;
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(dw_dtype == FAVAE_F32 || dw_dtype == dtype, "favae_linear_act_bwd: dw is fp32 or of the operands' type");
    FAVAE_CHECK_ARG(M == 0 || N == 0 || dy, "favae_linear_act_bwd: null dy");
    FAVAE_CHECK_ARG(!dx || K == 0 || N == 0 || w, "favae_linear_act_bwd: dx needs w");
    FAVAE_CHECK_ARG(!dw || K == 0 || M == 0 || x, "favae_linear_act_bwd: dw needs x");
    FAVAE_CHECK_ARG(act == FAVAE_ACT_NONE || M == 0 || N == 0 || pre, "favae_linear_act_bwd: the activation's gradient needs pre");
    FAVAE_CHECK_ARG(lddy >= N && (!x || ldx >= K) && (!w || ldw >= K) && (!pre || ldpre >= N) && (!dx || lddx >= K) && (!dw || lddw >= K) &&
                        (!xe || ldxe >= cdiv(K, CK_BLOCK)) && (!pe || ldpe >= cdiv(N, CK_BLOCK)),
                    "favae_linear_act_bwd: a row stride is below the row's length");
    FAVAE_CHECK_ARG(aligned(dy, es) && (xe || aligned(x, es)) && aligned(w, es) && (pe || aligned(pre, es)) && aligned(dx, es) &&
                        aligned(dw, dw_dtype == FAVAE_F32 ? 4 : 2),
                    "favae_linear_act_bwd: a pointer is not aligned to its type");
    const Operand od = {(const char*)dy, lddy, M, N}, ox = {(const char*)x, ldx, M, K}, ow = {(const char*)w, ldw, N, K};
    const int odd = std::max({odd_of(od, es), dx ? odd_of(ow, es) : 0, dw && !xe ? odd_of(ox, es) : 0});
    const BwdScratch sz = bwd_scratch(M, N, K, act, xe && dw, odd, es);
    FAVAE_CHECK_ARG(sz.total <= scratch_bytes && (sz.total == 0 || scratch) && aligned(scratch, 16), "favae_linear_act_bwd: scratch of %zu bytes, %zu needed",
                    scratch_bytes, sz.total);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == FAVAE_F32 ? lin_bwd<float>(od, ox, (const unsigned char*)xe, ldxe, ow, pre, ldpre, (const unsigned char*)pe, ldpe, M, N, K, act, dx, lddx,
                                               dw, lddw, 1, db, (char*)scratch, sz, st)
                              : lin_bwd<bf16_t>(od, ox, (const unsigned char*)xe, ldxe, ow, pre, ldpre, (const unsigned char*)pe, ldpe, M, N, K, act, dx, lddx,
                                                dw, lddw, dw_dtype == FAVAE_F32, db, (char*)scratch, sz, st);
}
