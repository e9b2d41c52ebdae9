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

typedef unsigned v4u __attribute__((ext_vector_type(4)));

struct GemmP {
    const char *P, *Q;                    // operands
    long long ldp, ldq;                   // elements
    const unsigned char* qe;              // exponents of Q where it is an 8-bit checkpoint
    long long ldqe;
    long long I, Cn;                      // output rows, reduction length
    int J;                                // output columns
    long long cchunk;                     // reduction elements of a split (a multiple of BK)
    int splits;
    int ti, tj;                           // tiles
    // output
    void* out; long long ldo;
    float* part;                          // splits > 1: [split][I][J]
    const float* bias;
    const void* res; long long ldr;
    void* pre; long long ldpre;
    int act;
    int vec;                              // out, res and pre allow 16-byte accesses of 8 columns
};


// LDS image of one operand's tile (ROWS outputs x BKE reduction elements of T).
//   KC: [ROWS][BKE], rows of 128 bytes (8 chunks of 16); chunk ^= (row >> 1) & 7: any 16 consecutive rows read at one chunk index cover the
//       256 bytes of a bank row once.
//   CM bf16: [BKE][ROWS]; the transposing load reads, per half wave, one 64-byte piece of 4 consecutive rows: the piece index is XORed
//       with row & 3 so that the four lie in different quarters of the 256-byte bank row.
//   CM fp32: [BKE][ROWS]; the two halves of a wave read rows k and k + 8: the 128-byte half is XORed with bit 3 of the row.
template <class T, int ROWS, bool CM> struct TileImg {
    static constexpr int BKE = 128 / sizeof(T);                       // 64 bf16, 32 fp32
    static constexpr int VE = 16 / sizeof(T);
    static constexpr int CPR = CM ? ROWS / VE : BKE / VE;             // chunks of a row
    static constexpr int CHUNKS = ROWS * BKE / VE;
    static constexpr int BYTES = CHUNKS * 16;
    __device__ static __forceinline__ int off(int row, int ch) {
        if constexpr (!CM) return row * 128 + ((ch ^ ((row >> 1) & 7)) << 4);
        else if constexpr (sizeof(T) == 2) return row * (ROWS * 2) + ((((ch >> 2) ^ (row & 3)) << 2 | (ch & 3)) << 4);
        else return row * (ROWS * 4) + ((ch ^ (row & 8)) << 4);
    }
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
            const int row = k0 + 8 * h + (i >> 2);                    // and row + 4: the same row & 3
            const int ch = ((((rb >> 5) ^ (row & 3)) << 2) | (2 * ((lane >> 4) & 1) + ((i & 3) >> 1)));
            const char* a = lds + row * (ROWS * 2) + ch * 16 + 8 * (i & 1);
            union { s16x4 s[2]; bf16x8 b; } c;
            c.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
            c.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 4 * ROWS * 2));
            f.v = c.b;
        } else {
            const int ch = (rb + r) >> 2;
#pragma unroll
            for (int j = 0; j < 8; ++j) f.v[j] = *(const float*)(lds + off(k0 + 8 * h + j, ch) + 4 * (r & 3));
        }
    }
};

// Staging of one operand's tile.  REG: through registers, any alignment, any tail; CKPT: the operand is an 8-bit checkpoint.
enum { S_REG = 0, S_CKPT = 1 };

template <class T, int ROWS, bool CM, int MODE, int NT> struct Stager {
    typedef TileImg<T, ROWS, CM> Img;
    static constexpr int NC = Img::CHUNKS / NT;
    static_assert(Img::CHUNKS % NT == 0, "whole chunks per thread");
    uint4 v[NC];
    // o0: first output row of the tile, no: output rows that exist; c0: first reduction element, cn: end of this split
    __device__ __forceinline__ void load(const GemmP& p, const char* base, long long ld, long long o0, long long no, long long c0, long long cn) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (int)threadIdx.x + i * NT, row = c / Img::CPR, ch = c - row * Img::CPR;
            // row / column position in memory: KC: rows are outputs; CM: rows are reduction elements
            const long long rr = (CM ? c0 : o0) + row, rn = CM ? cn : no;
            const long long cc = (CM ? o0 : c0) + ch * Img::VE, ce = CM ? no : cn;
            uint4 t = make_uint4(0u, 0u, 0u, 0u);
            if (rr < rn && cc < ce) {
                if constexpr (MODE == S_REG) {
                    const T* a = (const T*)base + rr * ld + cc;
                    if (cc + Img::VE <= ce) __builtin_memcpy(&t, a, 16);
                    else {
                        T tmp[Img::VE];
#pragma unroll
                        for (int j = 0; j < Img::VE; ++j) tmp[j] = cc + j < ce ? a[j] : (T)0;
                        __builtin_memcpy(&t, tmp, 16);
                    }
                } else {
                    const unsigned char* a = (const unsigned char*)base + rr * ld + cc;
                    unsigned w[2] = {0u, 0u};
                    if (cc + Img::VE <= ce) __builtin_memcpy(w, a, Img::VE);
                    else
#pragma unroll
                        for (int j = 0; j < Img::VE; ++j) if (cc + j < ce) w[j >> 2] |= (unsigned)a[j] << (8 * (j & 3));
                    t.x = w[0]; t.y = w[1];
                    t.z = p.qe[rr * p.ldqe + (cc >> 5)];
                }
            }
            v[i] = t;
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (int)threadIdx.x + i * NT, row = c / Img::CPR, ch = c - row * Img::CPR;
            uint4 t = v[i];
            if constexpr (MODE == S_CKPT) {
                const float s = ck_scale(t.z);
                if constexpr (sizeof(T) == 2) {
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = ck_byte(j < 4 ? t.x : t.y, j & 3) * s;
                    vec_put(t, f);
                } else {
                    float f[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[j] = ck_byte(t.x, j) * s;
                    t = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
                }
            }
            *(uint4*)(lds + Img::off(row, ch)) = t;
        }
    }
};

// 8 neighbouring output columns of one row: bias, activation, residual, store
template <class T, class OT> __device__ __forceinline__ void epilogue8(const GemmP& p, float (&f)[8], long long i, int j) {
    const int left = p.J - j;
    if (p.bias) {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] += k < left ? p.bias[j + k] : 0.f;
    }
    if (p.pre) {
        OT* o = (OT*)p.pre + i * p.ldpre + j;
        if (p.vec && left >= 8) {
            if constexpr (sizeof(OT) == 2) { uint4 r; vec_put(r, f); *(uint4*)o = r; }
            else { ((float4*)o)[0] = make_float4(f[0], f[1], f[2], f[3]); ((float4*)o)[1] = make_float4(f[4], f[5], f[6], f[7]); }
        } else
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k < left) o[k] = from_f32<OT>(f[k]);
    }
    act_apply<T>(f, p.act);
    if (p.res) {
        const T* a = (const T*)p.res + i * p.ldr + j;
        float t[8];
        if (p.vec && left >= 8) {
            if constexpr (sizeof(T) == 2) vec_get(t, *(const uint4*)a);
            else {
                const float4 lo = ((const float4*)a)[0], hi = ((const float4*)a)[1];
                t[0] = lo.x; t[1] = lo.y; t[2] = lo.z; t[3] = lo.w; t[4] = hi.x; t[5] = hi.y; t[6] = hi.z; t[7] = hi.w;
            }
        } else
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = k < left ? to_f32<T>(a[k]) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] += t[k];
    }
    OT* o = (OT*)p.out + i * p.ldo + j;
    if (p.vec && left >= 8) {
        if constexpr (sizeof(OT) == 2) { uint4 r; vec_put(r, f); *(uint4*)o = r; }
        else { ((float4*)o)[0] = make_float4(f[0], f[1], f[2], f[3]); ((float4*)o)[1] = make_float4(f[4], f[5], f[6], f[7]); }
    } else
#pragma unroll
        for (int k = 0; k < 8; ++k) if (k < left) o[k] = from_f32<OT>(f[k]);
}

// T: type of the operands and the residual, OT: of the output (and pre).  TI x TJ output tile, WI x WJ waves.
template <class T, class OT, int TI, int TJ, int WI, int WJ, bool PCM, bool QCM, int QMODE>
__global__ __launch_bounds__(64 * WI * WJ) void gemm_kernel(const GemmP p) {
    constexpr int NT = 64 * WI * WJ;
    typedef TileImg<T, TI, PCM> PI;
    typedef TileImg<T, TJ, QCM> QI;
    constexpr int BKE = PI::BKE, STAGE = PI::BYTES + QI::BYTES;
    constexpr int NI = TI / WI / 32, NJ = TJ / WJ / 32;
    extern __shared__ char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave / WJ, wj = wave - wi * WJ;
    // block -> (split, tile): blocks are dealt to the 8 XCDs in turn; each XCD takes a contiguous run of tiles, bands of 8 tile rows
    // walked column by column, so that the tiles running at one time share operand rows in one L2
    const long long n = (long long)p.ti * p.tj * p.splits, per = n / 8, b = blockIdx.x;
    long long lb = b < per * 8 ? (b & 7) * per + (b >> 3) : b;
    const int split = (int)(lb / ((long long)p.ti * p.tj));
    lb -= (long long)split * p.ti * p.tj;
    const int band = (int)(lb / (8 * p.tj)), in_band = (int)(lb - (long long)band * 8 * p.tj), bh = min(8, p.ti - band * 8);
    const int tj = in_band / bh, ti = band * 8 + in_band - tj * bh;
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

    Stager<T, TI, PCM, S_REG, NT> sp;
    Stager<T, TJ, QCM, QMODE, NT> sq;
    const int steps = (int)((ce - cb + BKE - 1) / BKE);
    if (steps > 0) {
        sp.load(p, p.P, p.ldp, i0, p.I, cb, ce);
        sq.load(p, p.Q, p.ldq, j0, p.J, cb, ce);
        sp.store(smem);
        sq.store(smem + PI::BYTES);
    }
    for (int t = 0; t < steps; ++t) {
        char* cur = smem + (t & 1) * STAGE;
        __syncthreads();
        if (t + 1 < steps) {
            sp.load(p, p.P, p.ldp, i0, p.I, cb + (long long)(t + 1) * BKE, ce);
            sq.load(p, p.Q, p.ldq, j0, p.J, cb + (long long)(t + 1) * BKE, ce);
        }
#pragma unroll
        for (int k = 0; k < BKE; k += 16) {
            Frag<T> fp[NI], fq[NJ];
#pragma unroll
            for (int a = 0; a < NI; ++a) PI::frag(fp[a], cur, wi * (TI / WI) + a * 32, k, lane);
#pragma unroll
            for (int c = 0; c < NJ; ++c) QI::frag(fq[c], cur + PI::BYTES, wj * (TJ / WJ) + c * 32, k, lane);
#pragma unroll
            for (int a = 0; a < NI; ++a)
#pragma unroll
                for (int c = 0; c < NJ; ++c) mma(acc[a][c], fq[c], fp[a]);
        }
        if (t + 1 < steps) {
            char* nxt = smem + ((t + 1) & 1) * STAGE;
            sp.store(nxt);
            sq.store(nxt + PI::BYTES);
        }
    }
    // epilogue: 32 output rows of the wave at a time through a region of LDS of its own, [32][NJ * 32 + 4] fp32, so that a lane ends up with 8 neighbouring columns
    __syncthreads();
    constexpr int WC = NJ * 32, RS = WC + 4, LPR = WC / 8;
    float* tile = (float*)smem + wave * 32 * RS;
#pragma unroll
    for (int a = 0; a < NI; ++a) {
#pragma unroll
        for (int c = 0; c < NJ; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *(float4*)(tile + (lane & 31) * RS + c * 32 + 8 * e + 4 * (lane >> 5)) = make_float4(acc[a][c][4 * e], acc[a][c][4 * e + 1], acc[a][c][4 * e + 2], acc[a][c][4 * e + 3]);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 32 * LPR / 64; ++e) {
            const int row = (lane + 64 * e) / LPR, cc = ((lane + 64 * e) - row * LPR) * 8;
            const float4 lo = *(const float4*)(tile + row * RS + cc), hi = *(const float4*)(tile + row * RS + cc + 4);
            float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            const long long i = i0 + wi * (TI / WI) + a * 32 + row;
            const int j = j0 + wj * WC + cc;
            if (i < p.I && j < p.J) {
                if (p.splits > 1) {
                    float* o = p.part + ((long long)split * p.I + i) * p.J + j;
#pragma unroll
                    for (int k = 0; k < 8; ++k) if (j + k < p.J) o[k] = f[k];
                } else epilogue8<T, OT>(p, f, i, j);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Sum of the splits, then the epilogue
template <class T, class OT> __global__ __launch_bounds__(256) void gemm_join_kernel(const GemmP p) {
    const int per_row = (p.J + 7) / 8;
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long i = t / per_row;
    const int j = (int)(t - i * per_row) * 8;
    if (i >= p.I) return;
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.f;
    for (int s = 0; s < p.splits; ++s) {
        const float* a = p.part + ((long long)s * p.I + i) * p.J + j;
#pragma unroll
        for (int k = 0; k < 8; ++k) if (j + k < p.J) f[k] += a[k];
    }
    epilogue8<T, OT>(p, f, i, j);
}

// ---- du = dy act'(u) and the column sums of du ---------------------------------------------------------------------------
// A block takes DU_COLS = 256 columns of a run of rows: lane = 4 columns, 4 rows at a time; column sums (fp32) of the unrounded du go to
// part[run][N].  du is rounded to T, the type of the matrix operands; with act == none it is dy itself and only the sums are taken.
struct DuP {
    const void* dy; long long lddy;
    const void* pre; long long ldpre;
    const unsigned char *pq, *pe; long long ldpe;
    void* du;                              // [M][N] contiguous
    float* part;                           // NULL: no sums
    long long M, rows;
    int N, act;
};
template <class T, int V, int SRC> __global__ __launch_bounds__(256) void act_bwd_kernel(const DuP p) {   // SRC: 0 no activation, 1 pre, 2 checkpoint
    __shared__ float red[4][64 * V];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int j = blockIdx.x * (64 * V) + lane * V;
    const long long r0 = (long long)blockIdx.y * p.rows, r1 = min(p.M, r0 + p.rows);
    float s[V];
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = 0.f;
    if (j < p.N) {
#pragma unroll 4
        for (long long i = r0 + w; i < r1; i += 4) {
            typename VecOf<T, V>::raw rd;
            float d[V];
            rd = *(const typename VecOf<T, V>::raw*)((const T*)p.dy + i * p.lddy + j);
            vec_get(d, rd);
            if constexpr (SRC > 0) {
                float z[V];
                if constexpr (SRC == 1) vec_get(z, *(const typename VecOf<T, V>::raw*)((const T*)p.pre + i * p.ldpre + j));
                else {
                    const float sc = ck_scale(p.pe[i * p.ldpe + (j >> 5)]);
                    const unsigned char* a = p.pq + i * p.ldpre + j;
                    unsigned wd[2] = {0u, 0u};
                    __builtin_memcpy(wd, a, V);
#pragma unroll
                    for (int k = 0; k < V; ++k) z[k] = ck_byte(wd[k >> 2], k & 3) * sc;
                }
                act_grad_mul<T>(d, z, p.act);
                vec_put(rd, d);
                *(typename VecOf<T, V>::raw*)((T*)p.du + i * (long long)p.N + j) = rd;
            }
#pragma unroll
            for (int k = 0; k < V; ++k) s[k] += d[k];
        }
    }
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
// Splits of the reduction: as many as bring the launch to about two blocks per CU, each at least 4 steps long
int plan_splits(long long I, int J, long long Cn, int es) {
    const long long tiles = cdivll(I, 128) * cdivll(J, 128), bke = 128 / es;
    if (tiles >= CUS) return 1;
    long long s = std::min((2 * CUS) / tiles, cdivll(Cn, 4 * bke));
    return (int)std::max<long long>(1, std::min<long long>(s, 256));
}
long long split_chunk(long long Cn, int splits, int es) {
    const long long bke = 128 / es;
    return cdivll(cdivll(Cn, bke), splits) * bke;
}

template <class T, class OT, bool PCM, bool QCM, int QMODE> int gemm_run(GemmP p, hipStream_t st) {
    if (p.I == 0 || p.J == 0) return FAVAE_OK;
    constexpr int es = sizeof(T);
    p.ti = (int)cdivll(p.I, 128);
    p.tj = cdiv(p.J, 128);
    p.splits = plan_splits(p.I, p.J, p.Cn, es);
    p.cchunk = split_chunk(p.Cn, p.splits, es);
    p.splits = (int)std::max<long long>(1, cdivll(p.Cn, std::max<long long>(1, p.cchunk)));
    p.vec = p.ldo % 8 == 0 && aligned(p.out, 16) && (!p.res || (p.ldr % 8 == 0 && aligned(p.res, 16))) && (!p.pre || (p.ldpre % 8 == 0 && aligned(p.pre, 16)));
    const long long blocks = (long long)p.ti * p.tj * p.splits;
    FAVAE_CHECK_ARG(blocks <= 0x7fffffffLL, "favae_linear_act: too many rows for one launch");
    constexpr size_t lds = std::max<size_t>(2 * (size_t)(TileImg<T, 128, PCM>::BYTES + TileImg<T, 128, QCM>::BYTES), 4 * 32 * (64 + 4) * 4);
    gemm_kernel<T, OT, 128, 128, 2, 2, PCM, QCM, QMODE><<<(unsigned)blocks, 256, lds, st>>>(p);
    FAVAE_LAUNCH_CHECK();
    if (p.splits > 1) {
        gemm_join_kernel<T, OT><<<(unsigned)cdivll(p.I * ((p.J + 7) / 8), 256), 256, 0, st>>>(p);
        FAVAE_LAUNCH_CHECK();
    }
    return FAVAE_OK;
}

size_t round256(size_t a) { return (a + 255) & ~(size_t)255; }
size_t split_bytes(long long I, int J, long long Cn, int es) {
    if (I == 0 || J == 0) return 0;
    const int s = plan_splits(I, J, Cn, es);
    return s > 1 ? round256((size_t)s * I * J * sizeof(float)) : 0;
}
constexpr int DU_RUNS = 256;
long long du_rows(long long M) { return std::max<long long>(16, cdivll(M, DU_RUNS)); }

int lin_sizes(const char* who, long long M, int N, int K, int act, int dtype) {
    FAVAE_CHECK_ARG(dtype == FAVAE_F32 || dtype == FAVAE_BF16, "%s: dtype is neither fp32 nor bf16", who);
    FAVAE_CHECK_ARG(act >= FAVAE_ACT_NONE && act <= FAVAE_ACT_GELU_TANH, "%s: unknown activation %d", who, act);
    FAVAE_CHECK_ARG(M >= 0 && N >= 0 && K >= 0 && M <= 0x7fffffffLL && N <= (1 << 24) && K <= (1 << 24), "%s: a size is negative or too large", who);
    return FAVAE_OK;
}

struct BwdScratch { size_t du, colp, split, total; };
BwdScratch bwd_scratch(long long M, int N, int K, int act, int dtype) {
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    BwdScratch s;
    s.du = act == FAVAE_ACT_NONE ? 0 : round256((size_t)M * N * es);
    s.colp = M > 0 ? round256((size_t)cdivll(M, du_rows(M)) * N * sizeof(float)) : 0;
    s.split = std::max(split_bytes(M, K, N, es), split_bytes(N, K, M, es));    // the two products run one after the other
    s.total = s.du + s.colp + s.split;
    return s;
}

template <class T> int lin_bwd(const void* dy, long long lddy, const void* x, long long ldx, const unsigned char* xe, long long ldxe, const void* w,
                               long long ldw, const void* pre, long long ldpre, const unsigned char* pe, long long ldpe, long long M, int N, int K,
                               int act, void* dx, long long lddx, void* dw, long long lddw, int dw_f32, float* db, char* scratch,
                               const BwdScratch& sz, hipStream_t st) {
    constexpr int es = sizeof(T);
    const T* du = (const T*)dy;
    long long lddu = lddy;
    float* colp = (float*)(scratch + sz.du);
    if (M > 0 && N > 0 && (act != FAVAE_ACT_NONE || db)) {
        DuP d = {dy, lddy, pre, ldpre, (const unsigned char*)pre, pe, ldpe, scratch, db ? colp : nullptr, M, du_rows(M), N, act};
        const int src = act == FAVAE_ACT_NONE ? 0 : pe ? 2 : 1;
        constexpr int VW = 16 / es;
        const bool wide = N % VW == 0 && lddy % VW == 0 && aligned(dy, 16) && (src != 1 || (ldpre % VW == 0 && aligned(pre, 16)));
        const int v = wide ? VW : 1;
        const dim3 g((unsigned)cdiv(N, 64 * v), (unsigned)cdivll(M, d.rows));
        if (wide) {
            if (src == 0) act_bwd_kernel<T, VW, 0><<<g, 256, 0, st>>>(d);
            else if (src == 1) act_bwd_kernel<T, VW, 1><<<g, 256, 0, st>>>(d);
            else act_bwd_kernel<T, VW, 2><<<g, 256, 0, st>>>(d);
        } else {
            if (src == 0) act_bwd_kernel<T, 1, 0><<<g, 256, 0, st>>>(d);
            else if (src == 1) act_bwd_kernel<T, 1, 1><<<g, 256, 0, st>>>(d);
            else act_bwd_kernel<T, 1, 2><<<g, 256, 0, st>>>(d);
        }
        FAVAE_LAUNCH_CHECK();
        if (act != FAVAE_ACT_NONE) { du = (const T*)scratch; lddu = N; }
    }
    if (db && N > 0) {
        col_join_kernel<<<cdiv(N, 16), 512, 0, st>>>(colp, M > 0 ? cdivll(M, du_rows(M)) : 0, N, db);
        FAVAE_LAUNCH_CHECK();
    }
    float* part = (float*)(scratch + sz.du + sz.colp);
    if (dx) {
        GemmP p = {};
        p.P = (const char*)du; p.ldp = lddu; p.Q = (const char*)w; p.ldq = ldw; p.I = M; p.J = K; p.Cn = N;
        p.out = dx; p.ldo = lddx; p.part = part; p.act = FAVAE_ACT_NONE;
        const int rc = gemm_run<T, T, false, true, S_REG>(p, st);
        if (rc != FAVAE_OK) return rc;
    }
    if (dw) {
        GemmP p = {};
        p.P = (const char*)du; p.ldp = lddu; p.Q = (const char*)x; p.ldq = ldx; p.qe = xe; p.ldqe = ldxe; p.I = N; p.J = K; p.Cn = M;
        p.out = dw; p.ldo = lddw; p.part = part; p.act = FAVAE_ACT_NONE;
        if constexpr (es == 2) {
            if (dw_f32) return xe ? gemm_run<T, float, true, true, S_CKPT>(p, st) : gemm_run<T, float, true, true, S_REG>(p, st);
        }
        return xe ? gemm_run<T, T, true, true, S_CKPT>(p, st) : gemm_run<T, T, true, true, S_REG>(p, st);
    }
    return FAVAE_OK;
}

}  // namespace

extern "C" size_t favae_linear_act_fwd_scratch(long long M, int N, int K, int dtype) {
    if (lin_sizes("favae_linear_act_fwd_scratch", M, N, K, FAVAE_ACT_NONE, dtype) != FAVAE_OK) return 0;
    return split_bytes(M, N, K, dtype == FAVAE_F32 ? 4 : 2);
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
    const size_t need = split_bytes(M, N, K, es);
    FAVAE_CHECK_ARG(need <= scratch_bytes && (need == 0 || scratch), "favae_linear_act_fwd: scratch of %zu bytes, %zu needed", scratch_bytes, need);
    GemmP p = {};
    p.P = (const char*)x; p.ldp = ldx; p.Q = (const char*)w; p.ldq = ldw; p.I = M; p.J = N; p.Cn = K;
    p.out = y; p.ldo = ldy; p.part = (float*)scratch; p.bias = bias; p.res = residual; p.ldr = ldr; p.pre = pre; p.ldpre = ldpre; p.act = act;
    return dtype == FAVAE_F32 ? gemm_run<float, float, false, false, S_REG>(p, (hipStream_t)stream)
                              : gemm_run<bf16_t, bf16_t, false, false, S_REG>(p, (hipStream_t)stream);
}

extern "C" size_t favae_linear_act_bwd_scratch(long long M, int N, int K, int act, int dtype) {
    if (lin_sizes("favae_linear_act_bwd_scratch", M, N, K, act, dtype) != FAVAE_OK) return 0;
    return bwd_scratch(M, N, K, act, dtype).total;
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
    const BwdScratch sz = bwd_scratch(M, N, K, act, dtype);
    FAVAE_CHECK_ARG(sz.total <= scratch_bytes && (sz.total == 0 || scratch) && aligned(scratch, 16), "favae_linear_act_bwd: scratch of %zu bytes, %zu needed",
                    scratch_bytes, sz.total);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == FAVAE_F32
               ? lin_bwd<float>(dy, lddy, x, ldx, (const unsigned char*)xe, ldxe, w, ldw, pre, ldpre, (const unsigned char*)pe, ldpe, M, N, K, act, dx,
                                lddx, dw, lddw, 1, db, (char*)scratch, sz, st)
               : lin_bwd<bf16_t>(dy, lddy, x, ldx, (const unsigned char*)xe, ldxe, w, ldw, pre, ldpre, (const unsigned char*)pe, ldpe, M, N, K, act, dx,
                                 lddx, dw, lddw, dw_dtype == FAVAE_F32, db, (char*)scratch, sz, st);
}
