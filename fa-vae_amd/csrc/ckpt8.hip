// Activation checkpoints in 8 bits: pack and unpack.
//
// q [R][C] int8 and one code byte per 32 channels of a row; the format is defined in act8.h.  Both directions are one pass over the
// data and bound by memory: pack reads 2 or 4 bytes a value and writes 33/32, unpack the reverse.  65536 x 1024 bf16 there and back 75 us, 5.4 TB/s.
#include "act8.h"

namespace {

struct CkP {
    const void* x; long long ldx;
    long long xn; unsigned S;            // pack, samples of S rows each that are not one run: stride of a sample (ldx: of a row in it)
    unsigned char* q; long long ldq;
    unsigned char* e; long long lde;
    void* out; long long ldo;
    long long R; int C, nb;              // nb = blocks of 32 channels in a row
};

// A lane takes 8 channels, 4 neighbouring lanes a block; lanes of a row's last block that lie past C are idle.  U vectors a thread, all
// loads issued before the first use.  Rows of any stride and alignment; TAIL: C is no multiple of 8.
template <class T> __device__ __forceinline__ void load8(float (&f)[8], const T* a, int nv) {
    if constexpr (sizeof(T) == 2) vec_get(f, load16(a, nv));
    else {
        float lo[4], hi[4];
        vec_get(lo, load16(a, nv));
        vec_get(hi, load16(a + 4, nv - 4));
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[j] = lo[j]; f[4 + j] = hi[j]; }
    }
}
struct CkPlace { long long row; int c, nv; };
template <bool TAIL> __device__ __forceinline__ CkPlace ck_place(const CkP& p, int u, long long row0, int off0) {
    const unsigned per_row = (unsigned)p.nb * 4u, t = (unsigned)(off0 + u * 256) + threadIdx.x, dr = t / per_row;
    CkPlace k;
    k.row = row0 + dr;
    k.c = (int)(t - dr * per_row) * 8;
    k.nv = k.row < p.R ? p.C - k.c : 0;
    if (!TAIL && k.nv > 0) k.nv = 8;
    return k;
}
// SAMPLES: x lies in samples of p.S rows, q and e in one run all the same
template <class T, int U, bool TAIL, bool SAMPLES> __global__ __launch_bounds__(256) void ck_pack_kernel(const CkP p) {
    const long long base = (long long)blockIdx.x * (256 * U), row0 = base / (p.nb * 4);
    const int off0 = (int)(base - row0 * (p.nb * 4));
    const long long n0 = SAMPLES ? row0 / p.S : 0;
    float f[U][8];
    CkPlace k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        k[u] = ck_place<TAIL>(p, u, row0, off0);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[u][j] = 0.f;
        long long off = k[u].row * p.ldx;
        if constexpr (SAMPLES) {                                 // (rows since the start of sample n0: below S + 256 + 1)
            const unsigned r = (unsigned)(k[u].row - n0 * p.S), dn = r / p.S;
            off = (n0 + dn) * p.xn + (long long)(r - dn * p.S) * p.ldx;
        }
        if (k[u].nv > 0) load8(f[u], (const T*)p.x + off + k[u].c, TAIL ? k[u].nv : 8);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        unsigned m = ck_amax(f[u]);
        m = max(m, (unsigned)__shfl_xor((int)m, 1, 64));
        m = max(m, (unsigned)__shfl_xor((int)m, 2, 64));
        const unsigned code = ck_code(m);
        unsigned w[2];
        ck_bytes(w, f[u], code);
        unsigned char* q = p.q + k[u].row * p.ldq + k[u].c;
        if (k[u].nv >= 8) __builtin_memcpy(q, w, 8);
        else if constexpr (TAIL)
#pragma unroll
            for (int j = 0; j < 8; ++j) if (j < k[u].nv) q[j] = (unsigned char)(w[j >> 2] >> (8 * (j & 3)));
        if (k[u].nv > 0 && (k[u].c & 31) == 0) p.e[k[u].row * p.lde + (k[u].c >> 5)] = (unsigned char)code;
    }
}

template <class T, int U, bool TAIL> __global__ __launch_bounds__(256) void ck_unpack_kernel(const CkP p) {
    const long long base = (long long)blockIdx.x * (256 * U), row0 = base / (p.nb * 4);
    const int off0 = (int)(base - row0 * (p.nb * 4));
    unsigned w[U][2], code[U];
    CkPlace k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        k[u] = ck_place<TAIL>(p, u, row0, off0);
        w[u][0] = w[u][1] = code[u] = 0u;
        if (k[u].nv > 0) {
            const unsigned char* q = p.q + k[u].row * p.ldq + k[u].c;
            if (!TAIL || k[u].nv >= 8) __builtin_memcpy(w[u], q, 8);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) if (j < k[u].nv) w[u][j >> 2] |= (unsigned)q[j] << (8 * (j & 3));
            code[u] = p.e[k[u].row * p.lde + (k[u].c >> 5)];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (k[u].nv <= 0) continue;
        const float s = ck_scale(code[u]);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = ck_value(w[u][j >> 2], j & 3, s);
        T* o = (T*)p.out + k[u].row * p.ldo + k[u].c;
        uint4 r;
        const int nv = TAIL ? k[u].nv : 8;
        if constexpr (sizeof(T) == 2) { vec_put(r, f); store16(o, r, nv); }
        else {
            const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
            vec_put(r, lo); store16(o, r, nv);
            vec_put(r, hi); store16(o + 4, r, nv - 4);
        }
    }
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

constexpr int U = 4;
// a launch has at most 2^31 - 1 blocks
template <class F> int launch_ck(long long blocks, const char* who, F&& f) {
    FAVAE_CHECK_ARG(blocks <= 0x7fffffffLL, "%s: too many rows for one launch", who);
    if (blocks > 0) f((unsigned)blocks);
    FAVAE_LAUNCH_CHECK();
    return FAVAE_OK;
}

}  // namespace

int ck_pack_samples(const void* x, long long xn, long long xs, long long N, long long S, int C, void* q, long long ldq, void* e, long long lde, int dtype,
                    hipStream_t st) {
    const int nb = cdiv(C, CK_BLOCK);
    const bool run = N == 1 || S == 1 || xn == S * xs;
    const CkP p = {x, S == 1 && N > 1 ? xn : xs, xn, (unsigned)S, (unsigned char*)q, ldq, (unsigned char*)e, lde, nullptr, 0, N * S, C, nb};
    return launch_ck(cdivll(p.R * nb * 4, 256 * U), "favae_ckpt8_pack", [&](unsigned g) {
        const auto go = [&](auto t, auto tail) {
            constexpr bool TAIL = decltype(tail)::value;
            if (run) ck_pack_kernel<decltype(t), U, TAIL, false><<<g, 256, 0, st>>>(p);
            else ck_pack_kernel<decltype(t), U, TAIL, true><<<g, 256, 0, st>>>(p);
        };
        if (dtype == FAVAE_F32) C % 8 ? go(0.f, std::true_type()) : go(0.f, std::false_type());
        else C % 8 ? go(bf16_t(0), std::true_type()) : go(bf16_t(0), std::false_type());
    });
}

extern "C" int favae_ckpt8_pack(const void* x, long long ldx, long long R, int C, void* q, long long ldq, void* e, long long lde, int dtype,
                                void* stream) {
    FAVAE_CHECK_ARG(R >= 0 && C >= 0 && (dtype == FAVAE_F32 || dtype == FAVAE_BF16), "favae_ckpt8_pack: bad sizes or dtype");
    if (R == 0 || C == 0) return FAVAE_OK;
    FAVAE_CHECK_ARG(C <= (1 << 28), "favae_ckpt8_pack: more than 2^28 channels");
    FAVAE_CHECK_ARG(x && q && e && ldx >= C && ldq >= C && lde >= cdiv(C, CK_BLOCK), "favae_ckpt8_pack: null pointer or a row stride below the row's length");
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(aligned(x, es), "favae_ckpt8_pack: x is not aligned to its type");
    return ck_pack_samples(x, 0, ldx, 1, R, C, q, ldq, e, lde, dtype, (hipStream_t)stream);
}

extern "C" int favae_ckpt8_unpack(const void* q, long long ldq, const void* e, long long lde, long long R, int C, void* out, long long ldo,
                                  int dtype, void* stream) {
    FAVAE_CHECK_ARG(R >= 0 && C >= 0 && (dtype == FAVAE_F32 || dtype == FAVAE_BF16), "favae_ckpt8_unpack: bad sizes or dtype");
    if (R == 0 || C == 0) return FAVAE_OK;
    const int nb = cdiv(C, CK_BLOCK);
    FAVAE_CHECK_ARG(out && q && e && ldo >= C && ldq >= C && lde >= nb, "favae_ckpt8_unpack: null pointer or a row stride below the row's length");
    FAVAE_CHECK_ARG(C <= (1 << 28), "favae_ckpt8_unpack: more than 2^28 channels");
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(aligned(out, es), "favae_ckpt8_unpack: out is not aligned to its type");
    CkP p = {nullptr, 0, 0, 0, (unsigned char*)q, ldq, (unsigned char*)e, lde, out, ldo, R, C, nb};
    const hipStream_t st = (hipStream_t)stream;
    return launch_ck(cdivll(R * nb * 4, 256 * U), "favae_ckpt8_unpack", [&](unsigned g) {
        if (dtype == FAVAE_F32) C % 8 ? ck_unpack_kernel<float, U, true><<<g, 256, 0, st>>>(p) : ck_unpack_kernel<float, U, false><<<g, 256, 0, st>>>(p);
        else C % 8 ? ck_unpack_kernel<bf16_t, U, true><<<g, 256, 0, st>>>(p) : ck_unpack_kernel<bf16_t, U, false><<<g, 256, 0, st>>>(p);
    });
}
